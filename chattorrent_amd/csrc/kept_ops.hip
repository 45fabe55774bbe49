// Operators that keep a chat's cache within a bound: attention that adds up
// what each row of the cache receives (cc_attend_weigh), and giving up the rows
// with the least of it (cc_kv_evict). The cache is common.h's (KV geometry),
// its marks a weight and a token number of each row of a (page, kv head).
#include "cache_dev.h"

// ================================================================== weigh ===
// With s = q . k / sqrt(D) in log2 units, p = 2^(s - M) and l = sum of p over
// the rows that a query row sees, out = sum p v / l, and a cache row's weight
// grows by the sum of p / l over query rows and heads.
//
// M need not be the largest score, only near it. It is a whole number, so what
// brings sums from one M to another is a power of two, exactly, and it stays as
// it is while no score passes it by more than P_ROOM; then it is the largest
// score rounded up. p is formed 2^P_SHIFT times as large, in one rounding, at
// most 2^14, for the f16 pairs that enter the P.V product. (Whether a score is
// that far above M is asked of their difference, which is exact where they are
// near: from 2^27 on f32 rounds M + P_ROOM.)
typedef float4_t float4_a4 __attribute__((aligned(4)));
constexpr float P_SHIFT = 6.0f, P_ROOM = 8.0f, P_UNSHIFT = 1.0f / 64.0f;
// From this M on a score is rounded before M is taken off, in k_weigh_many, which
// sums up l, and in k_weigh_sums alike: the largest score then does not miss M,
// and a column's p / l add up to 1. (Below it one fma does both. A column may be
// past it in one and not yet in the other, by its M so far or by its neighbours':
// the two p are then 2^-24 * 2^10 apart. Scores of this size, some 700 before
// log2(e), cost a call of many rows 5-7%: 2^20 in its place would be faster for
// them, and p 4% apart.)
constexpr float M_LARGE = 1024.0f;

// Between what a wave's lanes write to LDS and what other lanes of it read or
// write there: the wave's LDS instructions run in their order, and the compiler
// keeps it.
__device__ static inline void wave_lds() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
}

// The largest of a lane's value and those of the lanes 16, 32 and 48 away.
__device__ static inline float rows_max(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
    x = fmaxf(u2f(a[0]), u2f(a[1]));
    a = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
    return fmaxf(u2f(a[0]), u2f(a[1]));
}
__device__ static inline uint32_t rows_max(uint32_t x) {
    auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(a[0], a[1]);
    a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max(a[0], a[1]);
}
// Two values as f16 pairs (split_hilo2's), the remainder in one v_fma_mix each:
// x - (float)hi, exact.
__device__ static inline void split_mix2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    typedef float f2_t __attribute__((ext_vector_type(2)));
    asm("" : "+v"(x0), "+v"(x1));
    const f2_t x = {x0, x1};
    hi = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, half2_t));
    f2_t r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r[0]) : "v"(hi), "v"(x0));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r[1]) : "v"(hi), "v"(x1));
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, half2_t));
}

__device__ static inline float pow2_diff(float a, float b) {   // 2^(a - b) of whole numbers, 0 where a is -inf
    return a == -INFINITY ? 0.0f : ldexpf(1.0f, (int)fmaxf(a - b, -300.0f));
}

// A scale's bits, which order as it does (none is negative); 0 of one that is
// no finite number: the others' precision does not hang on it.
__device__ static inline uint32_t finite_bits(uint32_t b) { return b < 0x7f800000u ? b : 0u; }

struct WeighUnit {
    WeighJob jb;
    int head, tile, split, splits, tiles, pages;
};
__device__ static inline int weigh_job_at(const WeighJobs& jobs, int u, int WeighJob::*first) {
    int lo = 0, hi = jobs.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (jobs.j[mid].*first <= u) lo = mid;
        else hi = mid;
    }
    return lo;
}
__host__ __device__ static inline int weigh_pages(const WeighJob& j) { return (j.past + j.n - 1) / 64 + 1; }
__host__ __device__ static inline int weigh_tiles(const WeighJob& j, const WeighPlan& p) {
    return (j.n * p.group + 16 * p.subs - 1) / (16 * p.subs);
}
// A workgroup of the kernels that add up weights takes FINISH_PAGES pages of a
// (job, kv head); page0 and the stored scores count in whole workgroups.
__host__ __device__ static inline int page_room(int pages) { return (pages + FINISH_PAGES - 1) / FINISH_PAGES * FINISH_PAGES; }
// The unit of a workgroup: an XCD gets a run of them (op_work's reason).
__device__ static inline bool weigh_unit(const WeighJobs& jobs, const WeighPlan& p, WeighUnit& w) {
    const int per = (int)gridDim.x >> 3, u = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
    if (u >= jobs.units) return false;
    w.jb = jobs.j[weigh_job_at(jobs, u, &WeighJob::unit0)];
    w.pages = weigh_pages(w.jb);
    w.tiles = weigh_tiles(w.jb, p);
    w.splits = (w.pages + p.per - 1) / p.per;
    const int r = u - w.jb.unit0;
    if (p.subs > 1) {   // tiles that read the same pages run together
        w.tile = r % w.tiles;
        w.split = r / w.tiles % w.splits;
    } else {
        w.split = r % w.splits;
        w.tile = r / w.splits % w.tiles;
    }
    w.head = r / w.splits / w.tiles;
    return true;
}

// 8 channels of column `col` of a job's (kv head): its query row rotated to
// its position.
__device__ static inline void query8(const CacheDev& c, const AxesDev& axes, const WeighJob& jb, const WeighPlan& p, int head,
                                     int col, int d0, const float* __restrict__ q, int64_t ldq, float (&r)[8]) {
    const int i = col / p.group, h = head * p.group + col % p.group;
    const int64_t row = (int64_t)jb.row0 + i;
    const float* x = q + row * ldq + (size_t)h * c.D;
    if (axes.pos) rotated8_at(x, d0, c, axes, row, p.vec, r);
    else rotated8(x, d0, c.rope + (size_t)(jb.past + i) * c.rot, c.rot, p.vec, r);
}

// The power of two that brings a column's largest |q| to 2^3 .. 2^4, as its
// exponent's negative.
__device__ static inline int query_exponent(float qmax) { return max((int)(f2u(qmax) >> 23) - 127, -100) - 3; }
__device__ static inline float score_scale(int D, int eq) {
    return 1.4426950408889634f / sqrtf((float)D) * u2f((uint32_t)(127 + eq) << 23);
}

// 8 codes (biased) times a scale each, as an f16 pair: u * s - 128 * s is (u -
// 128) * s in one rounding. The scales are in 2^7 .. 2^8 where they are largest,
// so a value is below 2^15, and keeps 22 bits down to 2^-18 of that.
__device__ static inline void code_pair(uint32_t lo4, uint32_t hi4, const float (&s)[8], u32x4& hi, u32x4& lo) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const uint32_t w = e < 4 ? lo4 : hi4;
        const float x = __builtin_fmaf((float)((w >> (8 * (e & 3))) & 0xffu), s[e], -128.0f * s[e]);
        const float y = __builtin_fmaf((float)((w >> (8 * (e & 3) + 8)) & 0xffu), s[e + 1], -128.0f * s[e + 1]);
        uint32_t h, l;
        split_mix2(x, y, h, l);
        hi[e >> 1] = h;
        lo[e >> 1] = l;
    }
}
__device__ static inline void code_pair(uint32_t lo4, uint32_t hi4, float s, half8_t& hi, half8_t& lo) {
    const float sv[8] = {s, s, s, s, s, s, s, s};
    u32x4 h, l;
    code_pair(lo4, hi4, sv, h, l);
    hi = __builtin_bit_cast(half8_t, h);
    lo = __builtin_bit_cast(half8_t, l);
}
// The exponent of the largest of scales (bits), within what the pair's scale
// can be: times pair_down(e) a scale is at most 2^8.
__device__ static inline int pair_exponent(uint32_t top) { return max((int)(top >> 23) - 127, -112); }
__device__ static inline float pair_down(int e) { return u2f((uint32_t)(134 - e) << 23); }
// What a sum of a page's products of pairs takes to be a score: sc (score_scale)
// and the 2^7 that the keys were brought to. It stays a normal number, so that a
// masked -inf is still -inf behind it, and a sum of 0 still 0. (A sum is below
// 2^27: what the lower bound holds back is a score below 2^-99. Beyond the upper
// one products of the largest q and k pass 2^146.)
__device__ static inline float pair_score(float sc, int e) {
    return __builtin_amdgcn_fmed3f(ldexpf(sc, e - 7), 0x1p-126f, 0x1.fffffep127f);
}

// Of a page's scales, for the f16 pairs below: 16 bytes, the exponents of each
// group's largest V scale, of the largest K scale at PAIR_K, and at PAIR_BAD
// whether a V scale is no finite number.
constexpr int PAIR_K = 8, PAIR_BAD = 9;
// A piece of 16 columns' queries, rotated, by 256 threads, and their scales for
// the scores: f32 in x, 8 channels d0 of column h at query_at. Ends past a
// barrier.
template <int NG>
__device__ static inline int query_at(int h, int d0) { return h * 32 * NG + (d0 ^ 8 * (h & (NG == 2 ? 7 : 15))); }
template <int NG>
__device__ static inline void rotate_piece(const CacheDev& c, const AxesDev& axes, const WeighJob& jb, const WeighPlan& p, int head,
                                           int col0, const float* __restrict__ q, int64_t ldq, float* x, int* eq, float* sc) {
    constexpr int D = 32 * NG;
    const int tid = threadIdx.x, gt = min(16, jb.n * p.group - col0);
    for (int i = tid; i < 16 * (D / 8); i += 256) {
        const int h = i / (D / 8), d0 = 8 * (i & (D / 8 - 1)), at = query_at<NG>(h, d0);
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (h < gt) query8(c, axes, jb, p, head, col0 + h, d0, q, ldq, v);
        *(float4*)&x[at] = make_float4(v[0], v[1], v[2], v[3]);
        *(float4*)&x[at + 4] = make_float4(v[4], v[5], v[6], v[7]);
    }
    __syncthreads();
    // 16 threads a column
    float m = 0.0f;
    for (int d = tid & 15; d < D; d += 16) m = fmaxf(m, fabsf(x[(tid >> 4) * D + d]));
    for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
    if ((tid & 15) == 0) {
        eq[tid >> 4] = query_exponent(m);
        sc[tid >> 4] = score_scale(D, query_exponent(m));
    }
    __syncthreads();
}
// Of these, what lane `lane` feeds the matrix products of group g.
template <int NG>
__device__ static inline void query_pair(const float* x, const int* eq, int g, int lane, u32x4& hi, u32x4& lo) {
    const int h = lane & 15, at = query_at<NG>(h, 32 * g + 8 * (lane >> 4));
    const float down = u2f((uint32_t)(127 - eq[h]) << 23);
    const float4_t a = *(const float4_t*)&x[at] * down, b = *(const float4_t*)&x[at + 4] * down;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float4_t v = e < 2 ? a : b;
        uint32_t h2, l2;
        split_mix2(v[2 * (e & 1)], v[2 * (e & 1) + 1], h2, l2);
        hi[e] = h2;
        lo[e] = l2;
    }
}

// What comes before attention of more than 16 columns: the queries, rotated
// once, as the matrix products take them (a piece of 16 columns is [hi, lo]
// [NG][64 lanes] of 8 f16, and its scale for the scores 16 f32), then, for
// k_weigh_many, the exponents of the jobs' pages, a wave each. Bound by its
// chain of loads (job, position, rope table, query): 8 us for 16 x 8 verify
// rows of 24 heads of 256, 8.5 for 512 rows of 32 heads of 128. (In k_weigh_page,
// which does it itself for up to 16 columns, the verify rows' three pieces in
// every workgroup took 13 us more than here.)
template <int NG>
__global__ __launch_bounds__(256) void k_weigh_query(CacheDev c, WeighJobs jobs, WeighPlan p, AxesDev axes,
                                                     const float* __restrict__ q, int64_t ldq, uint8_t* __restrict__ ws) {
    constexpr int D = 32 * NG;
    __shared__ __align__(16) float x[16 * D];
    __shared__ int s_eq[16];
    const int tid = threadIdx.x, piece = blockIdx.x;
    if (piece >= jobs.joins) {
        const int lane = tid & 63, u = (piece - jobs.joins) * 4 + (tid >> 6);
        const WeighJob jb = jobs.j[weigh_job_at(jobs, u, &WeighJob::page0)];
        const int pages = weigh_pages(jb), room = page_room(pages), head = (u - jb.page0) / room, pg = (u - jb.page0) % room;
        if (pg >= pages) return;
        const uint32_t id = c.page_table[(size_t)jb.slot * c.max_pages + pg];
        if (id >= (uint32_t)c.n_pages) return;
        const int held = jb.past + jb.n - 64 * pg;   // of the page's rows
        const size_t at = ((size_t)id * c.nKV + head) * c.blk + 64 * D;
        const uint32_t *ks = (const uint32_t*)(c.k + at), *vs = (const uint32_t*)(c.v + at);
        const int vt = 16 * ((lane & 15) >> 2) + 4 * (lane >> 4) + (lane & 3);   // the row of V's entry `lane`
        uint32_t top = 0;
        bool bad = false;
        uint8_t* to = ws + p.exps + (size_t)u * 16;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            if (lane < held) top = max(top, finite_bits(ks[lane * NG + g]));
            uint32_t v = vt < held ? vs[((lane >> 4) * NG + g) * 16 + (lane & 15)] : 0u;
            bad = bad || v >= 0x7f800000u;
            v = row_max_u32(finite_bits(v));
            v = max(v, (uint32_t)__shfl_xor((int)v, 16));
            v = max(v, (uint32_t)__shfl_xor((int)v, 32));
            if (lane == 0) to[g] = (uint8_t)(int8_t)pair_exponent(v);
        }
        top = row_max_u32(top);
        top = max(top, (uint32_t)__shfl_xor((int)top, 16));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32));
        bad = __any(bad);
        if (lane == 0) {
            to[PAIR_K] = (uint8_t)(int8_t)pair_exponent(top);
            to[PAIR_BAD] = bad;
        }
        return;
    }
    const WeighJob jb = jobs.j[weigh_job_at(jobs, piece, &WeighJob::join0)];
    const int per_head = weigh_tiles(jb, p) * p.subs, r = piece - jb.join0;
    rotate_piece<NG>(c, axes, jb, p, r / per_head, r % per_head * 16, q, ldq, x, s_eq, (float*)(ws + p.qs) + (size_t)piece * 16);
    u32x4* to = (u32x4*)(ws + p.q) + (size_t)piece * 2 * NG * 64;
    for (int i = tid; i < NG * 64; i += 256) {
        u32x4 hi, lo;
        query_pair<NG>(x, s_eq, i >> 6, i & 63, hi, lo);
        to[i] = hi;
        to[NG * 64 + i] = lo;
    }
}

// Attention of up to 16 * CT columns over `per` pages, a page at a time by the
// whole workgroup: of S^T = K . Q^T each of the four waves makes a page's 16
// rows, of O^T += V^T . P^T a quarter of the channels, and P meets in LDS. So a
// wave loads and unpacks a quarter of the page's codes, straight into the
// registers that the matrix products read, and no code is unpacked twice. Keys
// are whole numbers in f16, scaled in f32 behind each group's product; values
// are f16 pairs relative to the largest scale so far of their group; queries
// and P are f16 pairs as well. While a page is at its second product the next
// one's codes are on their way.
// A page takes one barrier: each wave forms its P with the M it has, and the
// waves see each other's largest scores with each other's P. Where one of those
// passes M by more than P_ROOM, every wave forms its P anew from a new M.
//
// Where p.score_cols is set the scores stay in the workspace, [page][column][64]
// f32, for k_weigh_finish: 4 bytes a column and token beside the 2 * (D + D/8)
// that a token's K and V take.
//
// 32 chats of 2048 .. 16384 tokens, 5 heads of 128 a kv head: 127 us, 0.57 GB of
// K, V and scores at 4.5 TB/s (a copy: 5.0). One chat of 9000: 12, a chain of
// the query's loads and five pages a workgroup. 16 chats x 8 verify rows
// (48 columns), heads of 256: 69 us, 2.6 TB/s: vector instructions (codes to
// f16, P times V's scales as pairs, exp2) and waiting at 8 waves a CU.
template <int NG, int CT>
__global__ __launch_bounds__(256, 2) void k_weigh_page(CacheDev c, WeighJobs jobs, WeighPlan p, AxesDev axes,
                                                       const float* __restrict__ q, int64_t ldq, float* __restrict__ out,
                                                       int64_t ldo, uint8_t* __restrict__ ws) {
    constexpr int D = 32 * NG, DW = D / 64, GW = DW > 1 ? DW / 2 : 1;   // of a wave: 16-channel pieces, groups
    // Where V's scales go. Into P, which is then split for each group (48 vector instructions a lane, group and 16 columns) and
    // multiplies whole numbers, one instruction a code and two products; or into V, as f16 pairs, 5.5 a code and three.
    constexpr bool PS = NG > 2 ? CT <= 3 : CT == 1;
    constexpr int PB = 4 * CT * 64;   // P of a page: PS: f32 [CT][4][64] of a lane's rows; else fragments [hi, lo][2][CT][64]
    __shared__ u32x4 qf[CT][2][NG][64];
    __shared__ u32x4 pbuf[2 * PB];
    __shared__ float tops[2][4][CT][16];
    __shared__ float s_sc[CT][16];
    __shared__ __align__(16) float ksl[4][NG][16], vsl[4][GW][64];   // each wave's own scales
    __shared__ uint32_t ids[256];
    WeighUnit w;
    if (!weigh_unit(jobs, p, w)) return;
    const WeighJob& jb = w.jb;
    const int tid = threadIdx.x, lane = tid & 63, j4 = lane >> 4, l16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cols = jb.n * p.group;
    const int e0 = w.split * p.per, e1 = min(e0 + p.per, w.pages);
    const uint32_t* pt = c.page_table + (size_t)jb.slot * c.max_pages;

    // a page's codes and scales on their way
    constexpr int SK = NG > 4 ? 2 : 1;   // scales a lane: K's of (row, group) e = SK * lane + ..; V's of entry e % 64 of group e / 64
    u32x4 kr[NG / 2], vr[DW];
    uint32_t ksr[SK], vsr[SK];
    const int ke0 = (SK * lane) % (16 * NG), ve0 = (SK * lane) % (64 * GW);
    auto rsrc = [&](const uint8_t* pool, uint32_t id) {
        const bool ok = id < (uint32_t)c.n_pages;   // an index outside the cache reads as zero, and is masked
        return __builtin_amdgcn_make_buffer_rsrc((void*)(pool + (ok ? ((size_t)id * c.nKV + w.head) * c.blk : 0)), 0,
                                                 ok ? c.blk : 0, 0x00020000);
    };
    auto load_k = [&](uint32_t id) {
        const auto r = rsrc(c.k, id);
#pragma unroll
        for (int i = 0; i < NG / 2; i++)
            kr[i] = __builtin_amdgcn_raw_buffer_load_b128(r, (16 * wave + l16) * D + (D / 4) * j4 + 16 * i, 0, 0);
#pragma unroll
        for (int i = 0; i < SK; i++) ksr[i] = __builtin_amdgcn_raw_buffer_load_b32(r, 64 * D + (16 * wave * NG + ke0 + i) * 4, 0, 0);
    };
    auto load_v = [&](uint32_t id) {
        const auto r = rsrc(c.v, id);
#pragma unroll
        for (int i = 0; i < DW; i++)
            vr[i] = __builtin_amdgcn_raw_buffer_load_b128(r, (j4 * D + (wave * DW + i) * 16 + l16) * 16, 0, 0);
#pragma unroll
        for (int i = 0; i < SK; i++) {
            const int e = ve0 + i, g = (wave * DW) / 2 + (e >> 6);
            vsr[i] = __builtin_amdgcn_raw_buffer_load_b32(r, 64 * D + (((e >> 4 & 3) * NG + g) * 16 + (e & 15)) * 4, 0, 0);
        }
    };
    const uint32_t my_id = pt[min(e0 + tid, e1 - 1)];
    uint32_t id = __builtin_amdgcn_readfirstlane(pt[e0]);
    ids[tid] = my_id;
    load_k(id);
    load_v(id);

    if (CT == 1) {   // the queries rotated here: a launch less, for some 2 us of every workgroup's time
        __shared__ int s_eq[16];
        float* x = (float*)&qf[0][0][0][0];   // as many bytes as their pairs take
        rotate_piece<NG>(c, axes, jb, p, w.head, 0, q, ldq, x, s_eq, s_sc[0]);
        constexpr int N = (NG + 3) / 4;
        u32x4 hi[N], lo[N];
        const bool mine = NG >= 4 || wave < NG;
#pragma unroll
        for (int i = 0; i < N; i++)
            if (mine) query_pair<NG>(x, s_eq, 4 * i + wave, lane, hi[i], lo[i]);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++)
            if (mine) {
                qf[0][0][4 * i + wave][lane] = hi[i];
                qf[0][1][4 * i + wave][lane] = lo[i];
            }
    } else {
        const size_t piece0 = (size_t)jb.join0 + (size_t)w.head * p.subs;
        const u32x4* of = (const u32x4*)(ws + p.q) + piece0 * 2 * NG * 64;
        u32x4* to = &qf[0][0][0][0];
#pragma unroll
        for (int i = 0; i < CT * NG / 2; i++) to[256 * i + tid] = of[256 * i + tid];
        if (tid < 16 * CT) s_sc[tid >> 4][tid & 15] = ((const float*)(ws + p.qs))[piece0 * 16 + tid];
    }
    __syncthreads();
    float sc[CT], M[CT], lsum[CT];
    int my_last[CT];
    float4_t o[DW][CT];
    bool store[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const int col = 16 * ct + l16;
        sc[ct] = s_sc[ct][l16];
        M[ct] = -INFINITY;
        lsum[ct] = 0.0f;
        my_last[ct] = jb.past + min(col, cols - 1) / p.group;
        store[ct] = p.score_cols > 0 && col < cols && col >= jb.count0 * p.group;
#pragma unroll
        for (int i = 0; i < DW; i++) o[i][ct] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    int ev[GW];   // O of a group's channels is relative to 2^ev, or 2^(ev - 7) of pairs
#pragma unroll
    for (int g = 0; g < GW; g++) ev[g] = -112;
    float* score_at = (float*)(ws + p.scores) +
                      (((size_t)jb.page0 + (size_t)w.head * page_room(w.pages) + e0) * p.score_cols + l16) * 64 + 16 * wave + 4 * j4;
    for (int e = e0; e < e1; e++) {
        const int b = (e - e0) & 1, r0 = 64 * e + 16 * wave + 4 * j4;   // the lane's first row of S
        const bool ok = id < (uint32_t)c.n_pages;
        const uint32_t next = __builtin_amdgcn_readfirstlane(ids[min(e + 1, e1 - 1) - e0]);
        const bool edge = !ok || 64 * e + 63 > jb.past;    // a row that not every column sees
        float4_t s[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) s[ct] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < SK; i++) ksl[wave][(ke0 + i) % NG][(ke0 + i) / NG] = u2f(ksr[i]);
        wave_lds();
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const float4_t ks = *(const float4_t*)&ksl[wave][g][4 * j4];
            const u32x4 kw = kr[g >> 1];
            const half8_t kf = (g & 1) ? dequant8_biased(kw[2], kw[3]) : dequant8_biased(kw[0], kw[1]);
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                float4_t pp = {0.f, 0.f, 0.f, 0.f};
                pp = mfma16x16x32(kf, __builtin_bit_cast(half8_t, qf[ct][0][g][lane]), pp);
                pp = mfma16x16x32(kf, __builtin_bit_cast(half8_t, qf[ct][1][g][lane]), pp);
#pragma unroll
                for (int r = 0; r < 4; r++) s[ct][r] = __builtin_fmaf(ks[r], pp[r], s[ct][r]);
            }
            if (CT * NG >= 16 && (g & 1)) __builtin_amdgcn_sched_barrier(0);   // no more query fragments ahead than fit
        }
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            if (edge) {
                const int last = ok ? my_last[ct] : -1;
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (r0 + r > last) s[ct][r] = -INFINITY;
            }
            s[ct] = s[ct] * sc[ct];
            if (store[ct]) *(float4_t*)(score_at + 16 * ct * 64) = s[ct];
            const float m = rows_max(fmaxf(fmaxf(s[ct][0], s[ct][1]), fmaxf(s[ct][2], s[ct][3])));
            if (j4 == 0) tops[b][wave][ct][l16] = m;
        }
        score_at += p.score_cols * 64;
        // (behind the stores: loads and stores are waited for in the order in which they were issued, and what waits for V
        // then waits for none of these)
        __builtin_amdgcn_sched_barrier(0);
        load_k(next);
        float sum[CT];
        uint2* pw = (uint2*)(pbuf + b * PB);
        auto form = [&]() {   // P of the wave's rows, relative to M
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                const float m = M[ct] == -INFINITY ? 0.0f : M[ct];
                float pr[4];
#pragma unroll
                for (int r = 0; r < 4; r++) pr[r] = __builtin_amdgcn_exp2f(s[ct][r] - m + P_SHIFT);
                sum[ct] = (pr[0] + pr[1]) + (pr[2] + pr[3]);
                if (PS) {
                    ((float4_t*)pbuf)[b * PB + (ct * 4 + wave) * 64 + lane] = float4_t{pr[0], pr[1], pr[2], pr[3]};
                    continue;
                }
                uint2 h, l;
                split_mix2(pr[0], pr[1], h.x, l.x);
                split_mix2(pr[2], pr[3], h.y, l.y);
                pw[(((0 * 2 + (wave >> 1)) * CT + ct) * 64 + lane) * 2 + (wave & 1)] = h;
                pw[(((1 * 2 + (wave >> 1)) * CT + ct) * 64 + lane) * 2 + (wave & 1)] = l;
            }
        };
        form();
        __syncthreads();
        bool over = false;
        float Mn[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const float m = fmaxf(fmaxf(tops[b][0][ct][l16], tops[b][1][ct][l16]), fmaxf(tops[b][2][ct][l16], tops[b][3][ct][l16]));
            const bool mine = m - M[ct] > P_ROOM;
            Mn[ct] = mine ? ceilf(m) : M[ct];
            over = over || mine;
        }
        if (__any(over)) {   // the same in every wave
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                const float alpha = pow2_diff(M[ct], Mn[ct]);
                lsum[ct] *= alpha;
#pragma unroll
                for (int i = 0; i < DW; i++) o[i][ct] = o[i][ct] * alpha;
                M[ct] = Mn[ct];
            }
            form();
            __syncthreads();
        }
#pragma unroll
        for (int ct = 0; ct < CT; ct++) lsum[ct] += sum[ct];
        // V's scales, relative to the largest so far of their group
        bool bad = false;
#pragma unroll
        for (int i = 0; i < SK; i++) {
            const int v = ve0 + i, row = 64 * e + 16 * (v >> 2 & 3) + 4 * (v >> 4 & 3) + (v & 3);
            if (row >= jb.past + jb.n) vsr[i] = 0u;
            bad = bad || vsr[i] >= 0x7f800000u;
            vsr[i] = finite_bits(vsr[i]);
        }
        uint32_t most = row_max_u32(max(vsr[0], vsr[SK - 1]));   // (a row of 16 lanes is of one group)
        if (GW == 1) most = rows_max(most);
        else most = max(most, (uint32_t)__shfl_xor((int)most, 16));
#pragma unroll
        for (int g = 0; g < GW; g++) {
            const int en = max(ev[g], pair_exponent(__builtin_amdgcn_readlane(most, 32 * g)));
            if (en != ev[g]) {
                const float f = ldexpf(1.0f, max(ev[g] - en, -300));
#pragma unroll
                for (int i = 0; i < DW; i++)
                    if ((DW > 1 ? i >> 1 : 0) == g)
#pragma unroll
                        for (int ct = 0; ct < CT; ct++) o[i][ct] = o[i][ct] * f;
                ev[g] = en;
            }
        }
        const float down = pair_down(GW > 1 && lane >= 32 ? ev[GW - 1] : ev[0]) * (PS ? 1.0f / 128.0f : 1.0f);
#pragma unroll
        for (int i = 0; i < SK; i++) vsl[wave][(ve0 + i) >> 6][(ve0 + i) & 63] = u2f(vsr[i]) * down;
        wave_lds();
        auto scales8 = [&](int g, int ks, float (&s8)[8]) {   // of the lane's rows 16 * (2 ks + i / 4) + 4 * j4 + i % 4
            const float4_t sa = *(const float4_t*)&vsl[wave][g][16 * j4 + 8 * ks], sb = *(const float4_t*)&vsl[wave][g][16 * j4 + 8 * ks + 4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s8[i] = sa[i];
                s8[4 + i] = sb[i];
            }
        };
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            if (PS) {
                float4_t pa[CT], pb[CT];
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    pa[ct] = ((const float4_t*)pbuf)[b * PB + (ct * 4 + 2 * ks) * 64 + lane];
                    pb[ct] = ((const float4_t*)pbuf)[b * PB + (ct * 4 + 2 * ks + 1) * 64 + lane];
                }
#pragma unroll
                for (int g = 0; g < GW; g++) {
                    float s8[8];
                    scales8(g, ks, s8);
                    half8_t vf[2];
#pragma unroll
                    for (int i = 0; i < (DW > 1 ? 2 : 1); i++) vf[i] = dequant8_biased(vr[2 * g + i][2 * ks], vr[2 * g + i][2 * ks + 1]);
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        u32x4 h4, l4;
#pragma unroll
                        for (int i = 0; i < 8; i += 2) {
                            const float4_t pv = i < 4 ? pa[ct] : pb[ct];
                            uint32_t h, l;
                            split_mix2(pv[i & 3] * s8[i], pv[(i & 3) + 1] * s8[i + 1], h, l);
                            h4[i >> 1] = h;
                            l4[i >> 1] = l;
                        }
                        const half8_t ph = __builtin_bit_cast(half8_t, h4), pl = __builtin_bit_cast(half8_t, l4);
#pragma unroll
                        for (int i = 0; i < (DW > 1 ? 2 : 1); i++) {
                            o[2 * g + i][ct] = mfma16x16x32(vf[i], ph, o[2 * g + i][ct]);
                            o[2 * g + i][ct] = mfma16x16x32(vf[i], pl, o[2 * g + i][ct]);
                        }
                    }
                }
                continue;
            }
            half8_t ph[CT], pl[CT];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                ph[ct] = __builtin_bit_cast(half8_t, pbuf[b * PB + (0 * 2 + ks) * CT * 64 + ct * 64 + lane]);
                pl[ct] = __builtin_bit_cast(half8_t, pbuf[b * PB + (1 * 2 + ks) * CT * 64 + ct * 64 + lane]);
            }
#pragma unroll
            for (int i = 0; i < DW; i++) {
                float s8[8];
                scales8(DW > 1 ? i >> 1 : 0, ks, s8);
                u32x4 h, l;
                code_pair(vr[i][2 * ks], vr[i][2 * ks + 1], s8, h, l);
                const half8_t vh = __builtin_bit_cast(half8_t, h), vl = __builtin_bit_cast(half8_t, l);
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    o[i][ct] = mfma16x16x32(vh, ph[ct], o[i][ct]);
                    o[i][ct] = mfma16x16x32(vl, ph[ct], o[i][ct]);
                    o[i][ct] = mfma16x16x32(vh, pl[ct], o[i][ct]);
                }
                if (CT * NG >= 16 && (i & 1)) __builtin_amdgcn_sched_barrier(0);
            }
        }
        load_v(next);
        if (ok && __any(bad)) {   // a scale that is no finite number: NaN for the columns that see it
            const uint32_t* vs = (const uint32_t*)(c.v + ((size_t)id * c.nKV + w.head) * c.blk + 64 * D);
#pragma unroll
            for (int g = 0; g < GW; g++)
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    int any = 0;
                    for (int i = 0; i < 16; i++)   // entry i: row 16 * (i / 4) + 4 * j4 + i % 4
                        any |= 64 * e + 16 * (i >> 2) + 4 * j4 + (i & 3) <= my_last[ct] &&
                               vs[(j4 * NG + (wave * DW) / 2 + g) * 16 + i] >= 0x7f800000u;
                    any |= __shfl_xor(any, 16);
                    any |= __shfl_xor(any, 32);
                    if (any) {
#pragma unroll
                        for (int i = 0; i < DW; i++)
                            if ((DW > 1 ? i >> 1 : 0) == g)
#pragma unroll
                                for (int r = 0; r < 4; r++) o[i][ct][r] = NAN;
                    }
                }
        }
        id = next;
    }
    // l: a lane's rows, a wave's, the four waves'
    __syncthreads();
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        float l = lsum[ct] + __shfl_xor(lsum[ct], 16);
        l += __shfl_xor(l, 32);
        if (j4 == 0) tops[0][wave][ct][l16] = l;
    }
    __syncthreads();
    const size_t unit = (size_t)jb.unit0 + (size_t)w.head * w.splits + w.split;
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const int col = 16 * ct + l16;
        if (col >= cols) continue;
        const float l = ((tops[0][0][ct][l16] + tops[0][1][ct][l16]) + (tops[0][2][ct][l16] + tops[0][3][ct][l16])) * P_UNSHIFT;
        if (wave == 0 && j4 == 0) ((float2*)(ws + p.ml))[(unit * p.subs + ct) * 16 + l16] = make_float2(M[ct], l);
        float* part = (float*)(ws + p.parts) + ((unit * p.subs + ct) * 16 + l16) * D + wave * (D / 4) + 4 * j4;
        float* dst = out + ((int64_t)jb.row0 + col / p.group) * ldo + (size_t)(w.head * p.group + col % p.group) * D + wave * (D / 4) + 4 * j4;
#pragma unroll
        for (int i = 0; i < DW; i++) {
            float4_t y = o[i][ct] * ldexpf(P_UNSHIFT, ev[DW > 1 ? i >> 1 : 0] - (PS ? 0 : 7));
            if (w.splits == 1) {
#pragma unroll
                for (int r = 0; r < 4; r++) y[r] = l != 0.0f ? y[r] / l : 0.0f;
                *(float4_a4*)(dst + 16 * i) = y;
            } else {
                *(float4_t*)(part + 16 * i) = y;
            }
        }
    }
}

// M and l of a column over a unit's splits, dealt to the lane's row of 16
// (lane / 16 of four): at is the column's first (M, l), `stride` from one split
// to the next. Then over the four rows, in a fixed order.
__device__ static inline float2 column_total(const float2* __restrict__ at, int splits, int stride, int row) {
    float m = -INFINITY, l = 0.0f;
    for (int s0 = row; s0 < splits; s0 += 32) {
        float2 v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = s0 + 4 * i < splits ? at[(size_t)(s0 + 4 * i) * stride] : make_float2(-INFINITY, 0.0f);
        float mn = m;
#pragma unroll
        for (int i = 0; i < 8; i++) mn = fmaxf(mn, v[i].x);
        l *= pow2_diff(m, mn);
#pragma unroll
        for (int i = 0; i < 8; i++) l = __builtin_fmaf(v[i].y, pow2_diff(v[i].x, mn), l);
        m = mn;
    }
    const float mx = rows_max(m);
    l *= pow2_diff(m, mx);
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    return make_float2(mx, l);
}

// After k_weigh_page: joins the splits' outputs (the first workgroups, a
// WEIGH_JOIN floats of a 16-column piece each, its splits dealt to four waves)
// and, from the stored scores, adds up the weights of FINISH_PAGES pages of a
// (job, kv head) a workgroup, a row a lane. Loads in sequence (the columns' M and
// l; scores, ahead of these, 4 bytes a lane) and one exp2 a score: 4.5 us for one
// chat; 21 for 32 chats, the joins alone 10 (37 MB of scores, still in the
// last-level cache: 1.8 TB/s over the whole); 21 for verify rows (61 MB, 2.9
// TB/s). 4 and 16 pages a workgroup were slower.
template <int NG>
__global__ __launch_bounds__(256) void k_weigh_finish(CacheDev c, WeighJobs jobs, WeighPlan p, MarksDev marks,
                                                      float* __restrict__ out, int64_t ldo, const uint8_t* __restrict__ ws) {
    constexpr int D = 32 * NG, CH = 16 * D / WEIGH_JOIN;   // chunks of a 16-column piece
    __shared__ __align__(16) float4_t red[4][64];
    __shared__ float2 total[64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float2* ml = (const float2*)(ws + p.ml);
    if ((int)blockIdx.x < jobs.joins * CH) {
        const int piece = (int)blockIdx.x / CH, ch = (int)blockIdx.x % CH;
        const WeighJob jb = jobs.j[weigh_job_at(jobs, piece, &WeighJob::join0)];
        const int splits = (weigh_pages(jb) + p.per - 1) / p.per;
        if (splits == 1) return;   // the attention kernel wrote them
        const int r = piece - jb.join0, sub = r % p.subs, head = r / p.subs;
        const int gt = min(16, jb.n * p.group - sub * 16);
        const int h = (ch * WEIGH_JOIN + lane * 4) / D, d = (ch * WEIGH_JOIN + lane * 4) % D;
        if (ch * WEIGH_JOIN / D >= gt) return;
        const size_t unit = (size_t)jb.unit0 + (size_t)head * splits;
        if (wave == 0) {   // every column's M and l
            const float2 t = column_total(ml + (unit * p.subs + sub) * 16 + (lane & 15), splits, p.subs * 16, lane >> 4);
            if (lane < 16) total[lane] = t;
        }
        __syncthreads();
        const float2* at = ml + (unit * p.subs + sub) * 16 + h;
        const float4_t* part = (const float4_t*)(ws + p.parts) + ((unit * p.subs + sub) * 16 * D + ch * WEIGH_JOIN) / 4 + lane;
        const float m = total[h].x;
        float4_t x = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = wave; s0 < splits; s0 += 16) {
            float4_t y[4];
            float2 v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int s = min(s0 + 4 * i, splits - 1);
                v[i] = at[(size_t)s * p.subs * 16];
                y[i] = part[(size_t)s * p.subs * 4 * D];
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (s0 + 4 * i < splits && !(v[i].x == -INFINITY && v[i].y == 0.0f)) x += y[i] * pow2_diff(v[i].x, m);
        }
        red[wave][lane] = x;
        __syncthreads();
        if (wave || h >= gt) return;
        x = (x + red[1][lane]) + (red[2][lane] + red[3][lane]);
        const float l = total[h].y;
        const int col = sub * 16 + h;
        float* dst = out + ((int64_t)jb.row0 + col / p.group) * ldo + (size_t)(head * p.group + col % p.group) * D + d;
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = l != 0.0f ? x[e] / l : 0.0f;
        *(float4_a4*)dst = x;
        return;
    }
    const int u = ((int)blockIdx.x - jobs.joins * CH) * FINISH_PAGES;
    const WeighJob jb = jobs.j[weigh_job_at(jobs, u, &WeighJob::page0)];
    const int pages = weigh_pages(jb), room = page_room(pages);
    const int head = (u - jb.page0) / room, p0 = (u - jb.page0) % room;
    const int splits = (pages + p.per - 1) / p.per;
    const int c0 = jb.count0 * p.group, cols = jb.n * p.group;
    const size_t unit = (size_t)jb.unit0 + (size_t)head * splits;   // one tile a (job, kv head)
    // a wave's pages: what does not hang on the columns' totals is loaded before them
    constexpr int WP = FINISH_PAGES / 4;
    const float* s0 = (const float*)(ws + p.scores) + ((size_t)jb.page0 + (size_t)head * room + p0 + wave) * p.score_cols * 64 + lane;
    float x[WP][8], before[WP];
    float* wt[WP];
#pragma unroll
    for (int i = 0; i < WP; i++) {
        const int pg = p0 + wave + 4 * i, row = 64 * pg + lane;
        const uint32_t id = pg < pages ? c.page_table[(size_t)jb.slot * c.max_pages + pg] : 0xffffffffu;
        const bool there = id < (uint32_t)c.n_pages && row < jb.past + jb.n;
        wt[i] = there ? marks.weight + ((size_t)id * c.nKV + head) * 64 + lane : nullptr;
        before[i] = there && !(p.fade == 0.0f && row >= jb.fresh) ? *wt[i] : 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) x[i][e] = there ? s0[(size_t)(4 * i * p.score_cols + min(c0 + e, cols - 1)) * 64] : 0.0f;
    }
    if (wave < p.subs && 16 * wave < cols) {
        const int col = 16 * wave + (lane & 15);
        const float2 t = column_total(ml + unit * p.subs * 16 + col, splits, p.subs * 16, lane >> 4);
        if (lane < 16) total[col] = make_float2(t.x == -INFINITY ? 0.0f : t.x, t.y != 0.0f ? 1.0f / t.y : 0.0f);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WP; i++) {
        if (!wt[i]) continue;
        float got = 0.0f;
        const int sees = (64 * (p0 + wave + 4 * i) + lane - jb.past) * p.group;   // the first column that sees the lane's row
        auto add = [&](float x1, int col) {
            const float2 t = total[min(col, cols - 1)];
            // (p of one that does not is 0, but its 1/l may be NaN)
            if (col < cols) got = __builtin_fmaf(__builtin_amdgcn_exp2f(x1 - t.x), col >= sees ? t.y : 0.0f, got);
        };
#pragma unroll
        for (int e = 0; e < 8; e++) add(x[i][e], c0 + e);
        for (int col = c0 + 8; col < cols; col += 20) {
            float y[20];
#pragma unroll
            for (int e = 0; e < 20; e++) y[e] = s0[(size_t)(4 * i * p.score_cols + min(col + e, cols - 1)) * 64];
#pragma unroll
            for (int e = 0; e < 20; e++) add(y[e], col + e);
        }
        *wt[i] = __builtin_fmaf(before[i], 64 * (p0 + wave + 4 * i) + lane >= jb.fresh ? p.fade : 1.0f, got);   // weigh_add's sum
    }
}

// After k_weigh_many, where a tile's pages were split: joins the outputs of
// 1024 / D columns of a piece a workgroup, 4 channels a thread, and leaves the
// columns' M and 1/l. 512 rows of 40 heads of 128: 8.6 us, the parts read and
// the output written (three splits: 42 MB) at 4.9 TB/s, from the last-level
// cache.
template <int NG>
__global__ __launch_bounds__(256) void k_weigh_join(WeighJobs jobs, WeighPlan p, float* __restrict__ out, int64_t ldo,
                                                    uint8_t* __restrict__ ws) {
    constexpr int D = 32 * NG, CH = D / 64;
    const int piece = (int)blockIdx.x / CH, i = ((int)blockIdx.x % CH) * 256 + (int)threadIdx.x, h = 4 * i / D, d = 4 * i % D;
    const WeighJob jb = jobs.j[weigh_job_at(jobs, piece, &WeighJob::join0)];
    const int tiles = weigh_tiles(jb, p), splits = (weigh_pages(jb) + p.per - 1) / p.per;
    if (splits == 1) return;   // the attention kernel wrote them
    const int r = piece - jb.join0, sub = r % p.subs, tile = r / p.subs % tiles, head = r / p.subs / tiles;
    const int col = (tile * p.subs + sub) * 16 + h;
    if (col >= jb.n * p.group) return;
    const size_t unit = (size_t)jb.unit0 + ((size_t)head * tiles + tile) * splits;
    const float2* at = (const float2*)(ws + p.ml) + (unit * p.subs + sub) * 16 + h;
    const float4_t* part = (const float4_t*)(ws + p.parts) + (unit * p.subs + sub) * 4 * D + i;
    float m = -INFINITY, l = 0.0f;
    float4_t x = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < splits; s0 += 4) {
        float4_t y[4];
        float2 v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int s = min(s0 + e, splits - 1);
            v[e] = at[(size_t)s * p.subs * 16];
            y[e] = part[(size_t)s * p.subs * 4 * D];
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (s0 + e >= splits || (v[e].x == -INFINITY && v[e].y == 0.0f)) continue;   // nothing seen: there is no part
            const float mn = fmaxf(m, v[e].x), fa = pow2_diff(m, mn), fb = pow2_diff(v[e].x, mn);
            l = l * fa + v[e].y * fb;
            x = x * fa + y[e] * fb;
            m = mn;
        }
    }
    float* dst = out + ((int64_t)jb.row0 + col / p.group) * ldo + (size_t)(head * p.group + col % p.group) * D + d;
    if (p.tot && d == 0) ((float2*)(ws + p.tot))[(size_t)piece * 16 + h] = make_float2(m, l != 0.0f ? 1.0f / l : 0.0f);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = l != 0.0f ? x[e] / l : 0.0f;
    *(float4_a4*)dst = x;
}

// Schedules a block of N groups of P matrix products, each group behind two LDS
// reads of its operands, so that the reads are three groups ahead. (ID: one a block.)
template <int N, int P, int ID>
__device__ static inline void reads_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, 6, ID);
#pragma unroll
    for (int i = 0; i < N; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, P, ID);
        if (i + 3 < N) __builtin_amdgcn_sched_group_barrier(0x100, 2, ID);
    }
}

// Attention of a tile of 16 * CT columns for each of W waves over `per` pages.
// The workgroup unpacks a step of TOK rows once for all its columns, K and V as
// f16 pairs relative to the page's largest scales (V: the largest so far), in
// the order in which the matrix products read them: a fragment is 64 lanes of
// 16 bytes. Each product is then three: hi * hi, lo * hi and hi * lo, into one
// f32 sum, and nothing is scaled in between (a pair's two halves hold 22 bits).
// While a step is computed the next one is unpacked into the other buffer and
// the one after it is loaded.
// Bound by the matrix units and what stands between their products: 512 rows of
// 40 heads of 128 at 8192 take 258 us, 0.27 TFLOP with three products for one
// (1.04 PFLOP/s; a large f16 matmul of random values: 1.25), 32 heads at 4000
// 114 us.
// The matrix units are busy 45-50% of the time and the vector unit about as
// long, for the exp2s and pairs of P, with little of either beside the other.
// Steps of 64 rows, wave priorities and unpacking between the products were
// slower (300 us the last).
template <int NG, int CT, int W, int TOK>
__global__ __launch_bounds__(64 * W, 2) void k_weigh_many(CacheDev c, WeighJobs jobs, WeighPlan p, float* __restrict__ out,
                                                          int64_t ldo, uint8_t* __restrict__ ws) {
    constexpr int D = 32 * NG, DT = D / 16, TT = TOK / 16, KS = TOK / 32, HALVES = 64 / TOK;
    constexpr int NK = TT * NG / 2, NV = DT, NKW = (NK + W - 1) / W, NVW = (NV + W - 1) / W;   // unpacking, in pieces of a wave
    __shared__ u32x4 kbuf[2][2][TT][NG][64];
    __shared__ u32x4 vbuf[2][2][KS][DT][64];
    __shared__ uint32_t ids[256];
    __shared__ u32x4 exps[256];
    WeighUnit w;
    if (!weigh_unit(jobs, p, w)) return;
    const WeighJob& jb = w.jb;
    const int tid = threadIdx.x, lane = tid & 63, j4 = lane >> 4, l16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cols = jb.n * p.group, tcol = w.tile * 16 * p.subs, tile_end = min(tcol + 16 * p.subs, cols);
    const int tile_pages = (jb.past + (tile_end - 1) / p.group) / 64 + 1;
    const int e0 = w.split * p.per, e1 = min(e0 + p.per, tile_pages);
    const size_t unit = (size_t)jb.unit0 + ((size_t)w.head * w.tiles + w.tile) * w.splits + w.split;
    float2* ml = (float2*)(ws + p.ml) + unit * p.subs * 16;
    if (e0 >= e1) {   // the tile ends before these pages
        if (tid < 16 * p.subs) ml[tid] = make_float2(-INFINITY, 0.0f);
        return;
    }
    const uint32_t* pt = c.page_table + (size_t)jb.slot * c.max_pages;
    {   // the pages and their scales' exponents
        const u32x4* ex = (const u32x4*)(ws + p.exps) + (size_t)jb.page0 + (size_t)w.head * page_room(w.pages) + e0;
        for (int i = tid; i < e1 - e0; i += 64 * W) {
            ids[i] = pt[e0 + i];
            exps[i] = ex[i];
        }
    }
    const int held = jb.past + jb.n, steps = (e1 - e0) * HALVES;
    // byte i of a page's exponents (NG <= 8)
    struct Exps {
        uint32_t w[3];
        __device__ int at(int i) const { return (int)(int8_t)(w[i >> 2] >> (8 * (i & 3))); }
    };
    auto exps_of = [&](int pg) {
        const u32x4 x = exps[pg];
        return Exps{{(uint32_t)__builtin_amdgcn_readfirstlane(x[0]), (uint32_t)__builtin_amdgcn_readfirstlane(x[1]),
                     (uint32_t)__builtin_amdgcn_readfirstlane(x[2])}};
    };
    // the wave's queries
    const int wcol = tcol + wave * CT * 16;
    const bool busy = wcol < cols;
    const size_t piece0 = (size_t)jb.join0 + ((size_t)w.head * w.tiles + w.tile) * p.subs + wave * CT;
    half8_t qh[CT][NG], ql[CT][NG];
    float sc[CT];
    int my_last[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const u32x4* qf = (const u32x4*)(ws + p.q) + (piece0 + ct) * 2 * NG * 64 + lane;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            qh[ct][g] = __builtin_bit_cast(half8_t, qf[g * 64]);
            ql[ct][g] = __builtin_bit_cast(half8_t, qf[(NG + g) * 64]);
        }
        sc[ct] = ((const float*)(ws + p.qs))[(piece0 + ct) * 16 + l16];
        my_last[ct] = jb.past + min(wcol + 16 * ct + l16, cols - 1) / p.group;
    }
    const int first_last = jb.past + wcol / p.group;   // the least of the wave's columns'
    __syncthreads();

    // a step's codes and scales on their way: pieces of 16 rows x 64 channels of K, of 16 channels x TOK rows of V
    u32x4 kr[NKW], vr[NVW], vsr[NVW][TOK / 16];
    uint2 ksr[NKW];
    const int at_k = l16 * D + (D / 4) * j4, at_ks = l16 * NG * 4, at_v = (j4 * D + l16) * 16, at_vs = j4 * NG * 64;
    auto load = [&](int st) {
        const uint32_t id = __builtin_amdgcn_readfirstlane(ids[st / HALVES]);
        const int half = st % HALVES;
        const bool ok = id < (uint32_t)c.n_pages;   // an index outside the cache reads as zero, and is masked
        const size_t at = ok ? ((size_t)id * c.nKV + w.head) * c.blk : 0;
        const auto rk = __builtin_amdgcn_make_buffer_rsrc((void*)(c.k + at), 0, ok ? c.blk : 0, 0x00020000);
        const auto rv = __builtin_amdgcn_make_buffer_rsrc((void*)(c.v + at), 0, ok ? c.blk : 0, 0x00020000);
#pragma unroll
        for (int k = 0; k < NKW; k++) {
            const int task = wave + W * k, t = half * TOK + 16 * (task / (NG / 2)), gp = task % (NG / 2);
            if (NK % W && task >= NK) break;
            kr[k] = __builtin_amdgcn_raw_buffer_load_b128(rk, at_k, t * D + 16 * gp, 0);
            const auto s2 = __builtin_amdgcn_raw_buffer_load_b64(rk, at_ks, 64 * D + (t * NG + 2 * gp) * 4, 0);
            ksr[k] = make_uint2(s2[0], s2[1]);
        }
#pragma unroll
        for (int k = 0; k < NVW; k++) {
            const int dt = wave + W * k;
            if (NV % W && dt >= NV) break;
            if (TOK == 64) vr[k] = __builtin_amdgcn_raw_buffer_load_b128(rv, at_v, dt * 256, 0);
            else {
                const auto x = __builtin_amdgcn_raw_buffer_load_b64(rv, at_v, dt * 256 + 8 * half, 0);
                vr[k][0] = x[0];
                vr[k][1] = x[1];
            }
#pragma unroll
            for (int i = 0; i < TOK / 16; i++)
                vsr[k][i] = __builtin_amdgcn_raw_buffer_load_b128(rv, at_vs, 64 * D + (dt >> 1) * 64 + 32 * half + 16 * i, 0);
        }
    };
    int etask[NVW];   // the largest V exponent so far of the pieces' groups
#pragma unroll
    for (int k = 0; k < NVW; k++) etask[k] = -112;
    auto unpack = [&](int st) {
        const int b = st & 1, half = st % HALVES, pg = st / HALVES;
        const int r0 = (e0 + pg) * 64 + half * TOK;   // the step's first row
        const Exps ex = exps_of(pg);
        const bool ok = __builtin_amdgcn_readfirstlane(ids[pg]) < (uint32_t)c.n_pages;
        const float kdown = ok ? pair_down(ex.at(PAIR_K)) : 0.0f;
#pragma unroll
        for (int k = 0; k < NKW; k++) {
            const int task = wave + W * k, tt = task / (NG / 2), gp = task % (NG / 2);
            if (NK % W && task >= NK) break;
            float s0 = u2f(ksr[k].x) * kdown, s1 = u2f(ksr[k].y) * kdown;
            if (r0 + TOK > held && r0 + 16 * tt + l16 >= held) s0 = s1 = 0.0f;
            half8_t h, l;
            code_pair(kr[k][0], kr[k][1], s0, h, l);
            kbuf[b][0][tt][2 * gp][lane] = __builtin_bit_cast(u32x4, h);
            kbuf[b][1][tt][2 * gp][lane] = __builtin_bit_cast(u32x4, l);
            code_pair(kr[k][2], kr[k][3], s1, h, l);
            kbuf[b][0][tt][2 * gp + 1][lane] = __builtin_bit_cast(u32x4, h);
            kbuf[b][1][tt][2 * gp + 1][lane] = __builtin_bit_cast(u32x4, l);
        }
#pragma unroll
        for (int k = 0; k < NVW; k++) {
            const int dt = wave + W * k;
            if (NV % W && dt >= NV) break;
            const int g = dt >> 1;
            if (ok) etask[k] = max(etask[k], (int)(int8_t)((g >= 4 ? ex.w[1] : ex.w[0]) >> (8 * (g & 3))));
            const float down = pair_down(etask[k]);
            float s[TOK / 4];
#pragma unroll
            for (int i = 0; i < TOK / 4; i++) s[i] = u2f(vsr[k][i >> 2][i & 3]) * down;
            if (ok && ex.at(PAIR_BAD)) {
#pragma unroll
                for (int i = 0; i < TOK / 4; i++) s[i] = u2f(finite_bits(vsr[k][i >> 2][i & 3])) * down;
            }
            if (r0 + TOK > held) {
#pragma unroll
                for (int i = 0; i < TOK / 4; i++)   // entry i: row 16 * (i / 4) + 4 * j4 + i % 4
                    if (r0 + 16 * (i >> 2) + 4 * j4 + (i & 3) >= held) s[i] = 0.0f;
            }
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const float s8[8] = {s[8 * ks], s[8 * ks + 1], s[8 * ks + 2], s[8 * ks + 3],
                                     s[8 * ks + 4], s[8 * ks + 5], s[8 * ks + 6], s[8 * ks + 7]};
                u32x4 h, l;
                code_pair(vr[k][2 * ks], vr[k][2 * ks + 1], s8, h, l);
                vbuf[b][0][ks][dt][lane] = h;
                vbuf[b][1][ks][dt][lane] = l;
            }
        }
    };

    float M[CT], lsum[CT], base[CT];
    bool large = false;   // an M of M_LARGE or more
    int ev[NG];   // O of a group's channels is relative to 2^(ev - 7)
    float4_t o[CT][DT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        M[ct] = -INFINITY;
        lsum[ct] = 0.0f;
        base[ct] = P_SHIFT;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[ct][dt] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int g = 0; g < NG; g++) ev[g] = -112;
    auto compute = [&](int st) {
        const int b = st & 1, half = st % HALVES, pg = st / HALVES;
        const int r0 = (e0 + pg) * 64 + half * TOK;
        const Exps ex = exps_of(pg);
        const bool ok = __builtin_amdgcn_readfirstlane(ids[pg]) < (uint32_t)c.n_pages;
        const int ke = ok ? ex.at(PAIR_K) : 0;
        float4_t acc[CT][TT];
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
#pragma unroll
            for (int tt = 0; tt < TT; tt++) acc[ct][tt] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int tt = 0; tt < TT; tt++) {
                const half8_t kh = __builtin_bit_cast(half8_t, kbuf[b][0][tt][g][lane]);
                const half8_t kl = __builtin_bit_cast(half8_t, kbuf[b][1][tt][g][lane]);
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    acc[ct][tt] = mfma16x16x32(kh, qh[ct][g], acc[ct][tt]);
                }
#pragma unroll
                for (int ct = 0; ct < CT; ct++) acc[ct][tt] = mfma16x16x32(kl, qh[ct][g], acc[ct][tt]);
#pragma unroll
                for (int ct = 0; ct < CT; ct++) acc[ct][tt] = mfma16x16x32(kh, ql[ct][g], acc[ct][tt]);
            }
        reads_ahead<NG * TT, 3 * CT, 0>();
        const bool edge = !ok || r0 + TOK - 1 > first_last;
        half8_t ph[CT][KS], pl[CT][KS];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const int last = ok ? my_last[ct] : -1;
            const float scp = pair_score(sc[ct], ke);
            if (edge) {
#pragma unroll
                for (int tt = 0; tt < TT; tt++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (r0 + 16 * tt + 4 * j4 + r > last) acc[ct][tt][r] = -INFINITY;
            }
            float top = -INFINITY;
#pragma unroll
            for (int tt = 0; tt < TT; tt++)
                top = fmaxf(fmaxf(top, fmaxf(acc[ct][tt][0], acc[ct][tt][1])), fmaxf(acc[ct][tt][2], acc[ct][tt][3]));
            top *= scp;
            if (__any(top - M[ct] > P_ROOM)) {   // (M -inf: the first score of a column)
                top = rows_max(top);
                const float Mn = top - M[ct] > P_ROOM ? ceilf(top) : M[ct];
                const float alpha = pow2_diff(M[ct], Mn);
                M[ct] = Mn;
                lsum[ct] *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) o[ct][dt] = o[ct][dt] * alpha;
                base[ct] = P_SHIFT - (Mn == -INFINITY ? 0.0f : Mn);
                large = __any(large || !(fabsf(base[ct]) < M_LARGE));
            }
            if (large) {
#pragma unroll
                for (int tt = 0; tt < TT; tt++)
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[ct][tt][r] = __builtin_amdgcn_exp2f(acc[ct][tt][r] * scp - (M[ct] == -INFINITY ? 0.0f : M[ct]) + P_SHIFT);
            } else {
#pragma unroll
                for (int tt = 0; tt < TT; tt++)
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[ct][tt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[ct][tt][r], scp, base[ct]));
            }
#pragma unroll
            for (int tt = 0; tt < TT; tt++) lsum[ct] += (acc[ct][tt][0] + acc[ct][tt][1]) + (acc[ct][tt][2] + acc[ct][tt][3]);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                u32x4 h4, l4;
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    uint32_t h, l;
                    split_mix2(acc[ct][2 * ks + (i >> 2)][i & 3], acc[ct][2 * ks + (i >> 2)][(i & 3) + 1], h, l);
                    h4[i >> 1] = h;
                    l4[i >> 1] = l;
                }
                ph[ct][ks] = __builtin_bit_cast(half8_t, h4);
                pl[ct][ks] = __builtin_bit_cast(half8_t, l4);
            }
        }
        int grown[NG];
        bool grew = false;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const int en = ok ? max(ev[g], ex.at(g)) : ev[g];
            grown[g] = ev[g] - en;
            grew = grew || grown[g];
            ev[g] = en;
        }
        if (grew) {
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int dt = 0; dt < DT; dt++) o[ct][dt] = o[ct][dt] * ldexpf(1.0f, max(grown[dt >> 1], -300));
        }
        if (ok && ex.at(PAIR_BAD)) {   // a V scale that is no finite number: NaN for the columns that see it
            const size_t at = ((size_t)__builtin_amdgcn_readfirstlane(ids[pg]) * c.nKV + w.head) * c.blk + 64 * D;
            const uint32_t* vs = (const uint32_t*)(c.v + at);
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    bool bad = false;
                    for (int i = 0; i < TOK / 4; i++) {
                        const int row = r0 + 16 * (i >> 2) + 4 * j4 + (i & 3);
                        if (row <= my_last[ct] && row < held && vs[(j4 * NG + g) * 16 + 8 * half * (TOK == 32) + i] >= 0x7f800000u) bad = true;
                    }
                    int any = bad;
                    any |= __shfl_xor(any, 16);
                    any |= __shfl_xor(any, 32);
                    if (any) {
#pragma unroll
                        for (int r = 0; r < 4; r++) o[ct][2 * g][r] = o[ct][2 * g + 1][r] = NAN;
                    }
                }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const half8_t vh = __builtin_bit_cast(half8_t, vbuf[b][0][ks][dt][lane]);
                const half8_t vl = __builtin_bit_cast(half8_t, vbuf[b][1][ks][dt][lane]);
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    o[ct][dt] = mfma16x16x32(vh, ph[ct][ks], o[ct][dt]);
                }
#pragma unroll
                for (int ct = 0; ct < CT; ct++) o[ct][dt] = mfma16x16x32(vl, ph[ct][ks], o[ct][dt]);
#pragma unroll
                for (int ct = 0; ct < CT; ct++) o[ct][dt] = mfma16x16x32(vh, pl[ct][ks], o[ct][dt]);
            }
        reads_ahead<KS * DT, 3 * CT, 1>();
    };
    load(0);
    unpack(0);
    if (steps > 1) load(1);
    __syncthreads();
    // half of the waves unpack before they compute and half after, so that a SIMD's two are not at their matrix products,
    // nor at the rest, at the same time
    const bool early = wave < W / 2;
    for (int st = 0; st < steps; st++) {
        auto ahead = [&]() {
            if (st + 1 < steps) unpack(st + 1);
            if (st + 2 < steps) load(st + 2);
        };
        if (early) ahead();
        if (busy) compute(st);
        if (!early) ahead();
        __syncthreads();
    }
    if (!busy) return;
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        lsum[ct] += __shfl_xor(lsum[ct], 16);
        lsum[ct] += __shfl_xor(lsum[ct], 32);
        const float l = lsum[ct] * P_UNSHIFT;
        const int col = wcol + 16 * ct + l16;
        if (col >= cols) continue;
        const int sub = wave * CT + ct;
        if (j4 == 0) {
            ml[sub * 16 + l16] = make_float2(M[ct], l);
            if (p.tot && w.splits == 1)
                ((float2*)(ws + p.tot))[(piece0 + ct) * 16 + l16] = make_float2(M[ct], l != 0.0f ? 1.0f / l : 0.0f);
        }
        float* part = (float*)(ws + p.parts) + ((unit * p.subs + sub) * 16 + l16) * D + 4 * j4;
        float* dst = out + ((int64_t)jb.row0 + col / p.group) * ldo + (size_t)(w.head * p.group + col % p.group) * D + 4 * j4;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            float4_t x = o[ct][dt] * ldexpf(P_UNSHIFT, ev[dt >> 1] - 7);
            if (w.splits == 1) {
#pragma unroll
                for (int r = 0; r < 4; r++) x[r] = l != 0.0f ? x[r] / l : 0.0f;
                *(float4_a4*)(dst + 16 * dt) = x;
            } else {
                *(float4_t*)(part + 16 * dt) = x;
            }
        }
    }
}

// The weights from many columns: q . k again, with the columns' M and l known.
// A wave holds the keys of 16 * TT rows of the cache as f16 pairs in registers
// and walks the columns of its chunk, a piece of 16 at a time, which its
// workgroup's four waves share through LDS; a lane adds up its 4 * TT rows' p /
// l, and 16 lanes meet at the end, in a fixed order. With one chunk the result
// goes to the marks, else to the chunk's line in the workspace (k_weigh_add).
// Three products as above: all 512 rows of 40 heads at 8192 counting 138 us
// (0.96 PFLOP/s), the last 64 of 512 rows of 32 heads at 4000 16. (Scores kept
// from the attention would be 0.7 GB of the former, written and read: 275 us.)
__device__ static inline void weigh_add(float* at, const WeighPlan& p, bool fades, float got) {
    const float before = fades && p.fade == 0.0f ? 0.0f : *at;
    *at = __builtin_fmaf(before, fades ? p.fade : 1.0f, got);
}
template <int NG>
__global__ __launch_bounds__(256, 2) void k_weigh_sums(CacheDev c, WeighJobs jobs, WeighPlan p, MarksDev marks,
                                                       uint8_t* __restrict__ ws) {
    constexpr int D = 32 * NG, TT = NG > 4 ? 2 : 4, PER_PAGE = 4 / TT, NQ = NG / 2;   // NQ: 16 bytes a thread of a piece
    __shared__ u32x4 qs[2][2 * NG * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, j4 = lane >> 4, l16 = lane & 15;
    constexpr int WGS = FINISH_PAGES * PER_PAGE / 4;   // workgroups of FINISH_PAGES pages
    const int u = (int)blockIdx.x / WGS * FINISH_PAGES;
    const WeighJob jb = jobs.j[weigh_job_at(jobs, u, &WeighJob::page0)];
    if (jb.count0 >= jb.n) return;   // a piece of a job before the rows that count
    const int pages = weigh_pages(jb), room = page_room(pages), head = (u - jb.page0) / room;
    const int part0 = (u - jb.page0) % room * PER_PAGE + (int)blockIdx.x % WGS * 4;   // the workgroup's first: 16 * TT rows each
    if (part0 / PER_PAGE >= pages) return;
    const int part = part0 + wave, pg = part / PER_PAGE, r0 = part * 16 * TT;     // the first of the wave's rows
    const uint32_t id = pg < pages ? c.page_table[(size_t)jb.slot * c.max_pages + pg] : 0xffffffffu;
    const bool busy = id < (uint32_t)c.n_pages;
    const int held = jb.past + jb.n, tiles = weigh_tiles(jb, p);
    const int c0 = jb.count0 * p.group, cols = jb.n * p.group;
    // the chunk's pieces, from the first whose columns see one of the workgroup's rows
    const int t0 = c0 / 16, t1 = (cols + 15) / 16, step = (t1 - t0 + p.chunks - 1) / p.chunks;
    const int to = min(t0 + ((int)blockIdx.y + 1) * step, t1);
    const int from = max(t0 + (int)blockIdx.y * step, max(c0, max(0, part0 * 16 * TT - jb.past) * p.group) / 16);
    const int my_from = busy ? max(0, r0 - jb.past) * p.group / 16 : to;
    const size_t piece0 = (size_t)jb.join0 + (size_t)head * tiles * p.subs;
    float4_t got[TT];
#pragma unroll
    for (int tt = 0; tt < TT; tt++) got[tt] = float4_t{0.f, 0.f, 0.f, 0.f};
    u32x4 qn[NQ];
    float2 tn;
    float scn;
    auto load = [&](int t16) {
        const u32x4* of = (const u32x4*)(ws + p.q) + (piece0 + t16) * 2 * NG * 64;
#pragma unroll
        for (int i = 0; i < NQ; i++) qn[i] = of[256 * i + tid];
        const int col = t16 * 16 + l16;
        tn = col < cols ? ((const float2*)(ws + p.tot))[(piece0 + t16) * 16 + l16] : make_float2(-INFINITY, 0.0f);
        scn = ((const float*)(ws + p.qs))[(piece0 + t16) * 16 + l16];
    };
    if (from < to) {
        load(from);
        half8_t kh[TT][NG], kl[TT][NG];
        // (a wave without a page goes through page 0's keys, for nothing)
        const uint8_t* blk = c.k + ((size_t)(busy ? id : 0u) * c.nKV + head) * c.blk;
        const int e = busy ? (int8_t)ws[p.exps + (size_t)(jb.page0 + head * room + pg) * 16 + PAIR_K] : 0;
        const float down = pair_down(e);
#pragma unroll
        for (int tt = 0; tt < TT; tt++) {
            const int r = r0 + 16 * tt + l16;
            const float* at = (const float*)(blk + 64 * D) + (r & 63) * NG;
#pragma unroll
            for (int g = 0; g < NG; g += 2) {
                const u32x4 w = *(const u32x4*)(blk + (size_t)(r & 63) * D + (D / 4) * j4 + 8 * g);
                const float2 sc = *(const float2*)(at + g);
                code_pair(w[0], w[1], r < held ? sc.x * down : 0.0f, kh[tt][g], kl[tt][g]);
                code_pair(w[2], w[3], r < held ? sc.y * down : 0.0f, kh[tt][g + 1], kl[tt][g + 1]);
            }
        }
        for (int t16 = from; t16 < to; t16++) {
            const int b = t16 & 1;
#pragma unroll
            for (int i = 0; i < NQ; i++) qs[b][256 * i + tid] = qn[i];
            const float2 t = tn;
            const float sc = pair_score(scn, e);
            __syncthreads();   // (a piece's place is written again two pieces on, past the next barrier)
            if (t16 + 1 < to) load(t16 + 1);
            if (t16 < my_from) continue;
            float4_t acc[TT];
#pragma unroll
            for (int tt = 0; tt < TT; tt++) acc[tt] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const half8_t qh = __builtin_bit_cast(half8_t, qs[b][g * 64 + lane]);
                const half8_t ql = __builtin_bit_cast(half8_t, qs[b][(NG + g) * 64 + lane]);
#pragma unroll
                for (int tt = 0; tt < TT; tt++) acc[tt] = mfma16x16x32(kh[tt][g], qh, acc[tt]);
#pragma unroll
                for (int tt = 0; tt < TT; tt++) acc[tt] = mfma16x16x32(kl[tt][g], qh, acc[tt]);
#pragma unroll
                for (int tt = 0; tt < TT; tt++) acc[tt] = mfma16x16x32(kh[tt][g], ql, acc[tt]);
            }
            const float base = t.x == -INFINITY ? 0.0f : -t.x;
            const bool large = __any(!(fabsf(base) < M_LARGE));
            const bool edge = t16 * 16 < c0 || t16 * 16 + 16 > cols || jb.past + t16 * 16 / p.group < r0 + 16 * TT - 1;
            if (!large && !edge) {
#pragma unroll
                for (int tt = 0; tt < TT; tt++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        got[tt][r] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(acc[tt][r], sc, base)), t.y, got[tt][r]);
                continue;
            }
            const int col = t16 * 16 + l16, last = col >= c0 && col < cols ? jb.past + col / p.group : -1;
#pragma unroll
            for (int tt = 0; tt < TT; tt++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float a = large ? acc[tt][r] * sc + base : __builtin_fmaf(acc[tt][r], sc, base);
                    const bool sees = r0 + 16 * tt + 4 * j4 + r <= last;
                    const float x = __builtin_amdgcn_exp2f(a);
                    got[tt][r] = __builtin_fmaf(sees ? x : 0.0f, sees ? t.y : 0.0f, got[tt][r]);
                }
        }
    }
    if (!busy) return;
#pragma unroll
    for (int tt = 0; tt < TT; tt++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            for (int o = 1; o < 16; o <<= 1) got[tt][r] += __shfl_xor(got[tt][r], o);
    if (l16) return;
    float* wt = marks.weight + ((size_t)id * c.nKV + head) * 64;
    float4_t* line = (float4_t*)(ws + p.lines) + (((size_t)blockIdx.y * jobs.pages + jb.page0 + head * room + pg) * 64 + (r0 & 63) + 4 * j4) / 4;
#pragma unroll
    for (int tt = 0; tt < TT; tt++) {
        if (p.chunks > 1) {
            line[4 * tt] = got[tt];
            continue;
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int row = r0 + 16 * tt + 4 * j4 + r;
            if (row < held) weigh_add(&wt[row & 63], p, row >= jb.fresh, got[tt][r]);
        }
    }
}

// The chunks' lines, added in their order: 5 us, a launch's time.
__global__ __launch_bounds__(256) static void k_weigh_add(CacheDev c, WeighJobs jobs, WeighPlan p, MarksDev marks,
                                                          const uint8_t* __restrict__ ws) {
    const int u = (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const WeighJob jb = jobs.j[weigh_job_at(jobs, u, &WeighJob::page0)];
    const int pages = weigh_pages(jb), room = page_room(pages), head = (u - jb.page0) / room, pg = (u - jb.page0) % room;
    if (jb.count0 >= jb.n || pg >= pages || 64 * pg + lane >= jb.past + jb.n) return;
    const uint32_t id = c.page_table[(size_t)jb.slot * c.max_pages + pg];
    if (id >= (uint32_t)c.n_pages) return;
    const float* line = (const float*)(ws + p.lines) + (size_t)u * 64 + lane;
    float got = 0.0f;
#pragma unroll 4
    for (int i = 0; i < p.chunks; i++) got += line[(size_t)i * jobs.pages * 64];
    weigh_add(marks.weight + ((size_t)id * c.nKV + head) * 64 + lane, p, 64 * pg + lane >= jb.fresh, got);
}

template <int NG>
static hipError_t weigh_ng(hipStream_t st, const CacheDev& c, const WeighJobs& jobs, const WeighPlan& p, WeighKind kind,
                           const AxesDev& axes, const MarksDev& marks, const float* q, int64_t ldq, float* out, int64_t ldo,
                           uint8_t* ws) {
    constexpr int D = 32 * NG, CH = 16 * D / WEIGH_JOIN, PER_PAGE = NG > 4 ? 2 : 1;
    const dim3 units(op_blocks(jobs.units));
    hipError_t e = hipSuccess;
    if (kind != WEIGH_FEW) {
        const int before = jobs.joins + (kind == WEIGH_WIDE ? jobs.pages / 4 : 0);
        e = op_launch(k_weigh_query<NG>, dim3(before), dim3(256), st, c, jobs, p, axes, q, ldq, ws);
        if (e != hipSuccess) return e;
    }
    auto page = [&](auto k) { return op_launch(k, units, dim3(256), st, c, jobs, p, axes, q, ldq, out, ldo, ws); };
    if (kind != WEIGH_WIDE) {
        if (p.subs == 1) e = page(k_weigh_page<NG, 1>);
        else if (p.subs == 2) e = page(k_weigh_page<NG, 2>);
        else if (p.subs == 3) e = page(k_weigh_page<NG, 3>);
        else e = page(k_weigh_page<NG, 4>);
    } else {
        e = op_launch(k_weigh_many<NG, (NG > 4 ? 1 : 2), 8, (NG > 2 ? 32 : 64)>, units, dim3(512), st, c, jobs, p, out, ldo, ws);
    }
    bool split = false;
    for (int j = 0; j < jobs.n; j++) split = split || weigh_pages(jobs.j[j]) > p.per;
    if (kind != WEIGH_WIDE) {
        WeighJobs finish = jobs;
        if (!split) finish.joins = 0;
        const int blocks = finish.joins * CH + (p.weigh ? jobs.pages / FINISH_PAGES : 0);
        if (e == hipSuccess && blocks)
            e = op_launch(k_weigh_finish<NG>, dim3(blocks), dim3(256), st, c, finish, p, marks, out, ldo, ws);
        return e;
    }
    if (e == hipSuccess && split) e = op_launch(k_weigh_join<NG>, dim3(jobs.joins * (D / 64)), dim3(256), st, jobs, p, out, ldo, ws);
    if (e == hipSuccess && p.weigh)
        e = op_launch(k_weigh_sums<NG>, dim3(jobs.pages * PER_PAGE / 4, p.chunks), dim3(256), st, c, jobs, p, marks, ws);
    if (e == hipSuccess && p.weigh && p.chunks > 1)
        e = op_launch(k_weigh_add, dim3(jobs.pages / 4), dim3(256), st, c, jobs, p, marks, ws);
    return e;
}

hipError_t launch_weigh(hipStream_t st, const CacheDev& c, const WeighJobs& jobs, const WeighPlan& plan, WeighKind kind,
                        const AxesDev& axes, const MarksDev& marks, const float* q, int64_t ldq, float* out, int64_t ldo,
                        uint8_t* ws) {
    WeighPlan p = plan;
    p.vec = aligned16(q) && aligned16(c.rope) && ldq % 4 == 0 && c.rot % 16 == 0;
    if (c.ng == 2) return weigh_ng<2>(st, c, jobs, p, kind, axes, marks, q, ldq, out, ldo, ws);
    if (c.ng == 4) return weigh_ng<4>(st, c, jobs, p, kind, axes, marks, q, ldq, out, ldo, ws);
    return weigh_ng<8>(st, c, jobs, p, kind, axes, marks, q, ldq, out, ldo, ws);
}

// ================================================================== evict ===
// What a row is kept by: its weight's order-preserving bits (-0 as 0; one that
// is no number counts least), above every weight where its token is one of the
// chat's first or latest.
__device__ static inline uint32_t keep_key(float weight, int token, int sink, int latest) {
    if (token < sink || token >= latest) return 0xffffffffu;
    return weight != weight ? 0u : order_bits(weight + 0.0f);
}

// Where a move's two rows lie: their (page, kv head) blocks in the cache and
// their places in them. of_row < 0: none.
struct EvictMove {
    uint32_t of, to;
    int of_row, to_row;
};

// The codes, scales and marks of N rows at a time, by a wave: all N are loaded
// before the first is stored (one after another a row waits for its page, its
// codes and the row before it). For the few moves of one workgroup; where a page
// gets many, k_evict_move.
template <int NG, int N>
__device__ static inline void move_rows(const CacheDev& c, const MarksDev& marks, const EvictMove* moves, int lane) {
    constexpr int D = 32 * NG, VB = D / 64;
    uint32_t kc[N], ks[N], vs[N], mk[N];
    uint8_t vc[N][VB];
    const int kl = min(lane, D / 4 - 1), gl = min(lane, NG - 1);
    const uint32_t* mark = lane & 1 ? (const uint32_t*)marks.token : (const uint32_t*)marks.weight;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const EvictMove m = moves[i];
        const int row = max(m.of_row, 0);
        const uint8_t *k = c.k + (size_t)m.of * c.blk, *v = c.v + (size_t)m.of * c.blk;
        kc[i] = *(const uint32_t*)(k + row * D + 4 * kl);
        ks[i] = *(const uint32_t*)(k + 64 * D + 4 * (row * NG + gl));
        vs[i] = *(const uint32_t*)(v + 64 * D + 4 * vscale_at(gl, row, NG));
        mk[i] = mark[(size_t)m.of * 64 + row];
#pragma unroll
        for (int e = 0; e < VB; e++) vc[i][e] = v[vcode_at(lane + 64 * e, row, D)];
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const EvictMove m = moves[i];
        if (m.of_row < 0) continue;
        uint8_t *k = c.k + (size_t)m.to * c.blk, *v = c.v + (size_t)m.to * c.blk;
        if (lane < D / 4) *(uint32_t*)(k + m.to_row * D + 4 * lane) = kc[i];
        if (lane < NG) {
            *(uint32_t*)(k + 64 * D + 4 * (m.to_row * NG + lane)) = ks[i];
            *(uint32_t*)(v + 64 * D + 4 * vscale_at(lane, m.to_row, NG)) = vs[i];
        }
        if (lane < 2) (lane ? (uint32_t*)marks.token : (uint32_t*)marks.weight)[(size_t)m.to * 64 + m.to_row] = mk[i];
#pragma unroll
        for (int e = 0; e < VB; e++) v[vcode_at(lane + 64 * e, m.to_row, D)] = vc[i][e];
    }
}
constexpr EvictMove NO_MOVE{0u, 0u, -1, -1};
__device__ static inline EvictMove move_at(const CacheDev& c, const uint32_t* pt, int head, int of, int to) {
    const uint32_t pf = pt[of >> 6], pg = pt[to >> 6];
    if (pf >= (uint32_t)c.n_pages || pg >= (uint32_t)c.n_pages) return NO_MOVE;
    return EvictMove{pf * (uint32_t)c.nKV + (uint32_t)head, pg * (uint32_t)c.nKV + (uint32_t)head, of & 63, to & 63};
}

// Sums of the lanes up to each, in six steps of the vector unit.
__device__ static inline uint32_t wave_running(uint32_t x) {
#define ADD_DPP(ctrl, rows) x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, false)
    ADD_DPP(0x111, 0xf);   // row_shr 1, 2, 4, 8
    ADD_DPP(0x112, 0xf);
    ADD_DPP(0x114, 0xf);
    ADD_DPP(0x118, 0xf);
    ADD_DPP(0x142, 0xa);   // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
    ADD_DPP(0x143, 0xc);
#undef ADD_DPP
    return x;
}

// A (job, kv head)'s list: the first move to each page below `keep`, their
// number, then (of, to) pairs.
__host__ __device__ static inline int evict_first(const EvictJob& j) { return ((j.keep + 63) / 64 + 2) & ~1; }
__device__ static inline int64_t evict_words(const EvictJob& j) { return evict_first(j) + 2 * (int64_t)j.room; }

// A workgroup of 1024 finds the rows that one (job, kv head) keeps. A thread
// holds a run of rows' keys (REG of them in registers; 0: as many as it takes,
// read again for each pass); the keep-th largest key comes from up to three
// passes over 11, 11 and 10 bits from the top with a histogram in LDS, the last
// one that where a digit's rows all stay; of its equals the lower rows stay.
// The rows below `keep` that go and the rows from `keep` on that stay are as
// many, and the i-th of the one takes the place of the i-th of the other: a
// list of them in the workspace, or up to EVICT_HERE moves made here.
// A chain of the keys' load, the passes' barriers and the list or the moves: 6
// us where one of 1025 rows goes, 20 where 32 chats of 4160 give up 64 each (9 of
// it before the moves), 16 for 16001 rows of one, 18 for 32 prompts of 2048 ..
// 16384.
template <int NG, int REG>
__global__ __launch_bounds__(1024) void k_evict_select(CacheDev c, EvictJobs jobs, MarksDev marks, int sink, int recent,
                                                       uint8_t* __restrict__ ws) {
    __shared__ uint32_t hist[3][2048];
    __shared__ uint32_t wsum[2][2][16];
    __shared__ uint32_t s_sel[3];
    __shared__ int here_rows[2 * EVICT_HERE];   // (of, to) pairs
    __shared__ EvictMove moves[EVICT_HERE];
    const EvictJob jb = jobs.j[blockIdx.x / c.nKV];
    const int head = (int)blockIdx.x % c.nKV;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const uint32_t* pt = c.page_table + (size_t)jb.slot * c.max_pages;
    const int latest = max(jb.seen - recent, 0);
    const int per = REG ? REG : (jb.rows + 4095) / 4096 * 4, i0 = min(t * per, jb.rows), i1 = min(i0 + per, jb.rows);
    auto key_at = [&](int i) -> uint32_t {
        const uint32_t pg = pt[i >> 6];
        if (pg >= (uint32_t)c.n_pages) return 0u;
        const size_t m = ((size_t)pg * c.nKV + head) * 64 + (i & 63);
        return keep_key(marks.weight[m], marks.token[m], sink, latest);
    };
    uint32_t reg[REG ? REG : 1];
    if (REG) {
        // a run of REG rows lies within a page
        const uint32_t pg = i0 < i1 ? pt[i0 >> 6] : 0xffffffffu;
        const bool ok = pg < (uint32_t)c.n_pages;
        const size_t m = ok ? ((size_t)pg * c.nKV + head) * 64 + (i0 & 63) : 0;
        float4 w[REG / 4 + 1];
        int4 k[REG / 4 + 1];
#pragma unroll
        for (int e = 0; e < REG / 4; e++) {
            w[e] = ok ? *(const float4*)(marks.weight + m + 4 * e) : make_float4(0.f, 0.f, 0.f, 0.f);
            k[e] = ok ? *(const int4*)(marks.token + m + 4 * e) : make_int4(0, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < REG / 4; e++) {
            reg[4 * e] = ok ? keep_key(w[e].x, k[e].x, sink, latest) : 0u;
            reg[4 * e + 1] = ok ? keep_key(w[e].y, k[e].y, sink, latest) : 0u;
            reg[4 * e + 2] = ok ? keep_key(w[e].z, k[e].z, sink, latest) : 0u;
            reg[4 * e + 3] = ok ? keep_key(w[e].w, k[e].w, sink, latest) : 0u;
        }
    }
    auto each = [&](auto&& f) {
        if (REG) {
#pragma unroll
            for (int e = 0; e < REG; e++)
                if (i0 + e < i1) f(i0 + e, reg[e]);
        } else {
            for (int i = i0; i < i1; i++) f(i, key_at(i));
        }
    };
    // what the threads before this one have of a, and all of them together; `turn` alternates from call to call
    auto before = [&](uint32_t a, int turn, int which, uint32_t& all) {
        const uint32_t x = wave_running(a);
        if (lane == 63) wsum[turn][which][wave] = x;
        __syncthreads();
        const uint32_t w = lane < 16 ? wsum[turn][which][lane] : 0u;
        const uint32_t r = wave_running(w);
        all = __builtin_amdgcn_readlane(r, 15);
        return x - a + (wave ? __builtin_amdgcn_readlane(r, wave - 1) : 0u);
    };
#pragma unroll
    for (int i = 0; i < 6; i++) ((uint32_t*)hist)[1024 * i + t] = 0;
    __syncthreads();
    uint32_t prefix = 0, left = (uint32_t)jb.keep, all = 0;
    bool every = false;   // every row with prefix's digits stays
#pragma unroll
    for (int ps = 0; ps < 3; ps++) {
        const int sh = ps == 0 ? 21 : ps == 1 ? 10 : 0, bits = ps == 2 ? 10 : 11;
        const uint32_t mask = (1u << bits) - 1;
        if (every) break;   // uniform
        each([&](int, uint32_t k) {
            if (ps == 0 || k >> (sh + bits) % 32 == prefix >> (sh + bits) % 32) atomicAdd(&hist[ps][(k >> sh) & mask], 1u);
        });
        __syncthreads();
        // thread t: the digits 2047 - 2t and 2046 - 2t, from the largest down
        const uint2 n = *(const uint2*)&hist[ps][2046 - 2 * t];
        const uint32_t b0 = before(n.x + n.y, ps & 1, 0, all);
        if (b0 < left && left <= b0 + n.x + n.y) {
            const bool first = left <= b0 + n.y;
            s_sel[0] = prefix | (uint32_t)(2047 - 2 * t - (first ? 0 : 1)) << sh;
            s_sel[1] = left - b0 - (first ? 0 : n.y);
            s_sel[2] = first ? n.y : n.x;
        }
        __syncthreads();
        prefix = s_sel[0];
        left = s_sel[1];
        every = s_sel[2] == left;
    }
    // every: the keys from `prefix` on stay; else `left` of those equal to it, and all above
    uint32_t eq = 0, be = 0;
    if (!every) {
        each([&](int, uint32_t k) { eq += k == prefix; });
        be = before(eq, 1, 0, all);
    }
    uint32_t to = 0, of = 0;
    const uint32_t be0 = be;
    auto kept = [&](uint32_t k) {
        if (every) return k >= prefix;
        const bool same = k == prefix, in = k > prefix || (same && be < left);
        be += same;
        return in;
    };
    each([&](int i, uint32_t k) {
        const bool in = kept(k), below = i < jb.keep;
        to += below && !in;
        of += !below && in;
    });
    uint32_t moved = 0;
    to = before(to, 0, 0, all);
    of = before(of, 0, 1, moved);
    be = be0;
    const bool here = jb.room <= EVICT_HERE;
    int32_t* list = (int32_t*)ws + jb.moves0 + (int64_t)head * evict_words(jb);
    int32_t* pairs = list + evict_first(jb);
    const int n = (int)min(moved, (uint32_t)jb.room);   // (within `room` unless another stream writes the marks meanwhile)
    if (!here && t == 0) list[(jb.keep + 63) >> 6] = n;
    each([&](int i, uint32_t k) {
        const bool in = kept(k);
        if (!here && i < jb.keep && (i & 63) == 0) list[i >> 6] = (int32_t)min(to, (uint32_t)n);
        const bool below = i < jb.keep, goes = below != in;
        const uint32_t at = below ? to : of;
        if (goes && at < (uint32_t)n) {
            if (here) here_rows[2 * at + below] = i;
            else pairs[2 * at + below] = i;
        }
        to += below && goes;
        of += !below && goes;
    });
    if (!here) return;
    __syncthreads();
    if (t < EVICT_HERE) moves[t] = t < n ? move_at(c, pt, head, here_rows[2 * t], here_rows[2 * t + 1]) : NO_MOVE;
    __syncthreads();
    if (4 * wave < n) move_rows<NG, 4>(c, marks, moves + 4 * wave, lane);   // 16 waves: EVICT_HERE
}
static_assert(EVICT_HERE == 64, "four moves for each of k_evict_select's sixteen waves");

// The moves of the lists: rows from `keep` on to rows below it, so no row is
// both read and written. A workgroup takes those to the rows of one (page, kv
// head). Where they are EVICT_PAGE or more, a thread takes a channel's 16 rows
// of V, whose codes lie beside each other, and puts the new ones into the 16
// bytes that it read; fewer are stored byte by byte.
// Bound by V's layout: a token's D codes lie in D/8 lines of 128 bytes, one in
// every 16 bytes, so a scattered row of V costs these lines, not D bytes. 32
// prompts (8 kv heads of 128) cut to 2048 rows: 122 us, 0.53 GB of lines at 4.3
// TB/s where the rows alone are 0.25 GB; one prompt of 4 heads of 256: 14 us.
constexpr int EVICT_PAGE = 8;
template <int NG>
__global__ __launch_bounds__(256) void k_evict_move(CacheDev c, EvictJobs jobs, MarksDev marks,
                                                    const uint8_t* __restrict__ ws) {
    constexpr int D = 32 * NG, DI = D / 64, SI = (NG + 3) / 4;   // 16 bytes of K or V a thread; scales
    __shared__ EvictMove moves[64];
    __shared__ int move_to[64];   // the move to a row of the page
    const EvictJob jb = jobs.j[blockIdx.y / c.nKV];
    const int head = (int)blockIdx.y % c.nKV, tid = threadIdx.x, pg = blockIdx.x;
    if (jb.room <= EVICT_HERE || 64 * pg >= jb.keep) return;
    const int32_t* list = (const int32_t*)ws + jb.moves0 + (int64_t)head * evict_words(jb);
    const int32_t* pairs = list + evict_first(jb);
    const int first = list[pg], n = min(list[pg + 1] - first, 64);
    if (n <= 0) return;
    const uint32_t* pt = c.page_table + (size_t)jb.slot * c.max_pages;
    if (tid < 64) {
        move_to[tid] = -1;
        wave_lds();      // (the 64 lanes of a wave)
        if (tid < n) {
            const int2 m = *(const int2*)(pairs + 2 * (first + tid));
            moves[tid] = move_at(c, pt, head, m.x, m.y);
            if (moves[tid].of_row >= 0) move_to[m.y & 63] = tid;
        }
    }
    __syncthreads();
    u32x4 kc[DI];
    uint32_t ks[SI], vs[SI], mark = 0;
#pragma unroll
    for (int e = 0; e < DI; e++) {
        const int i = 256 * e + tid, ch = i % (D / 16);
        const EvictMove m = moves[min(i / (D / 16), n - 1)];
        kc[e] = *(const u32x4*)(c.k + (size_t)m.of * c.blk + max(m.of_row, 0) * D + 16 * ch);
    }
#pragma unroll
    for (int e = 0; e < SI; e++) {
        const int i = 256 * e + tid, g = i % NG;
        const EvictMove m = moves[min(i / NG, n - 1)];
        const size_t at = (size_t)m.of * c.blk + 64 * D;
        ks[e] = *(const uint32_t*)(c.k + at + 4 * (max(m.of_row, 0) * NG + g));
        vs[e] = *(const uint32_t*)(c.v + at + 4 * vscale_at(g, max(m.of_row, 0), NG));
    }
    uint32_t* mark_of = tid & 1 ? (uint32_t*)marks.token : (uint32_t*)marks.weight;
    if (tid < 2 * n) mark = mark_of[(size_t)moves[tid >> 1].of * 64 + max(moves[tid >> 1].of_row, 0)];
    if (n >= EVICT_PAGE) {
        const uint32_t page = pt[pg];
        if (page < (uint32_t)c.n_pages) {
            u32x4* to = (u32x4*)(c.v + ((size_t)page * c.nKV + head) * c.blk);
#pragma unroll
            for (int e = 0; e < DI; e++) {
                const int i = 256 * e + tid, j4 = __builtin_amdgcn_readfirstlane(i / D), d = i % D;   // a wave's rows: 16 of the page
                u32x4 w = to[i];
                uint32_t b[16];
#pragma unroll
                for (int u = 0; u < 16; u++) {
                    const int at = __builtin_amdgcn_readfirstlane(move_to[16 * (u >> 2) + 4 * j4 + (u & 3)]);
                    b[u] = 0x100u;
                    if (at >= 0) b[u] = c.v[(size_t)moves[at].of * c.blk + vcode_at(d, moves[at].of_row, D)];
                }
#pragma unroll
                for (int u = 0; u < 16; u++) {
                    const uint32_t sh = 8 * (u & 3);
                    if (b[u] < 0x100u) w[u >> 2] = (w[u >> 2] & ~(0xffu << sh)) | b[u] << sh;
                }
                to[i] = w;
            }
        }
    } else {
        for (int i = tid; i < n * D; i += 256) {
            const EvictMove m = moves[i / D];
            if (m.of_row >= 0)
                c.v[(size_t)m.to * c.blk + vcode_at(i % D, m.to_row, D)] = c.v[(size_t)m.of * c.blk + vcode_at(i % D, m.of_row, D)];
        }
    }
#pragma unroll
    for (int e = 0; e < DI; e++) {
        const int i = 256 * e + tid, ch = i % (D / 16);
        const EvictMove m = moves[min(i / (D / 16), n - 1)];
        if (i < n * (D / 16) && m.of_row >= 0) *(u32x4*)(c.k + (size_t)m.to * c.blk + m.to_row * D + 16 * ch) = kc[e];
    }
#pragma unroll
    for (int e = 0; e < SI; e++) {
        const int i = 256 * e + tid, g = i % NG;
        const EvictMove m = moves[min(i / NG, n - 1)];
        if (i >= n * NG || m.of_row < 0) continue;
        const size_t at = (size_t)m.to * c.blk + 64 * D;
        *(uint32_t*)(c.k + at + 4 * (m.to_row * NG + g)) = ks[e];
        *(uint32_t*)(c.v + at + 4 * vscale_at(g, m.to_row, NG)) = vs[e];
    }
    if (tid < 2 * n && moves[tid >> 1].of_row >= 0) mark_of[(size_t)moves[tid >> 1].to * 64 + moves[tid >> 1].to_row] = mark;
}

template <int NG>
static hipError_t evict_ng(hipStream_t st, const CacheDev& c, const EvictJobs& jobs, int max_rows, const MarksDev& marks,
                           int sink, int recent, uint8_t* ws) {
    const dim3 grid(jobs.n * c.nKV);
    hipError_t e;
    if (max_rows <= 4096) e = op_launch(k_evict_select<NG, 4>, grid, dim3(1024), st, c, jobs, marks, sink, recent, ws);
    else if (max_rows <= 8192) e = op_launch(k_evict_select<NG, 8>, grid, dim3(1024), st, c, jobs, marks, sink, recent, ws);
    else if (max_rows <= 16384) e = op_launch(k_evict_select<NG, 16>, grid, dim3(1024), st, c, jobs, marks, sink, recent, ws);
    else e = op_launch(k_evict_select<NG, 0>, grid, dim3(1024), st, c, jobs, marks, sink, recent, ws);
    if (e == hipSuccess && jobs.room > EVICT_HERE)
        e = op_launch(k_evict_move<NG>, dim3((jobs.keep + 63) / 64, jobs.n * c.nKV), dim3(256), st, c, jobs, marks, ws);
    return e;
}

size_t evict_list_words(const EvictJob& j) { return evict_first(j) + 2 * (size_t)j.room; }

hipError_t launch_evict(hipStream_t st, const CacheDev& c, const EvictJobs& jobs, int max_rows, const MarksDev& marks,
                        int sink, int recent, uint8_t* ws) {
    if (c.ng == 2) return evict_ng<2>(st, c, jobs, max_rows, marks, sink, recent, ws);
    if (c.ng == 4) return evict_ng<4>(st, c, jobs, max_rows, marks, sink, recent, ws);
    return evict_ng<8>(st, c, jobs, max_rows, marks, sink, recent, ws);
}
