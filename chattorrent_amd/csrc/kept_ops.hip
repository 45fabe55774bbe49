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
// M need not be the largest score, only near it: it is the largest rounded up
// to a whole number. So what brings sums from one M to another is a power of
// two, exactly, and p can be formed 2^14 times as large, in one rounding, for
// the f16 pairs that enter the P.V product (p to 2^-24 of 2^14 there).
constexpr float P_SHIFT = 14.0f, P_UNSHIFT = 1.0f / 16384.0f;
constexpr float M_LARGE = 1048576.0f;   // beyond: the score is rounded before M is taken off, or the largest may miss it

__device__ static inline float pow2_diff(float a, float b) {   // 2^(a - b) of whole numbers, 0 where a is -inf
    return a == -INFINITY ? 0.0f : ldexpf(1.0f, (int)fmaxf(a - b, -300.0f));
}

constexpr int FINISH_PAGES = 8;

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
    w.split = r % w.splits;
    w.tile = r / w.splits % w.tiles;
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

// Attention of a tile of 16 columns over `per` pages, split over four waves. A
// wave walks its pages as attention over selected pages does (cache_ops.hip):
// S^T = K . Q^T with the query as an f16 pair, O^T += V^T . (p * s) with p * s
// as an f16 pair and V scales relative to their page and group's largest power
// of two; one page of codes in flight. Where p.score_cols is set the scores
// stay in the workspace, [page][column][64] f32, for k_weigh_finish: 4 bytes a
// column and token beside the 2 * (D + D/8) that a token's K and V take.
template <int NG>
__global__ __launch_bounds__(256, NG > 4 ? 1 : 2) void k_weigh(CacheDev c, WeighJobs jobs, WeighPlan p, AxesDev axes,
                                                               const float* __restrict__ q, int64_t ldq,
                                                               float* __restrict__ out, int64_t ldo,
                                                               uint8_t* __restrict__ ws) {
    constexpr int D = 32 * NG, DT = D / 16, SCL = NG > 4 ? NG / 4 : 1;
    constexpr int OW = 16 * D + 32;   // floats of a wave's part: O [16][D], M [16], l [16]
    __shared__ __align__(16) float smem[4 * OW];
    WeighUnit w;
    if (!weigh_unit(jobs, p, w)) return;
    const WeighJob& jb = w.jb;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, j4 = lane >> 4, l16 = lane & 15;
    const int col0 = w.tile * 16, gt = min(16, jb.n * p.group - col0);
    const int e0 = w.split * p.per, e1 = min(e0 + p.per, w.pages);
    const uint32_t* pt = c.page_table + (size_t)jb.slot * c.max_pages;
    // this wave's pages, an index a lane (per <= 256)
    const int n = e1 - e0, w0 = e0 + (n * wave) / 4, nw = e0 + (n * (wave + 1)) / 4 - w0;
    const uint32_t pgv = lane < nw ? pt[w0 + lane] : 0u;
    for (int i = tid; i < gt * (D / 8); i += 256) {
        const int h = i / (D / 8), d0 = 8 * (i & (D / 8 - 1));
        float r[8];
        query8(c, axes, jb, p, w.head, col0 + h, d0, q, ldq, r);
        *(float4*)&smem[h * D + d0] = make_float4(r[0], r[1], r[2], r[3]);
        *(float4*)&smem[h * D + d0 + 4] = make_float4(r[4], r[5], r[6], r[7]);
    }
    __syncthreads();
    float qmax = 0.0f;
    const bool live = l16 < gt;
#pragma unroll
    for (int i = 0; i < 8 * NG; i += 4) {
        const float4 f = *(const float4*)&smem[l16 * D + 32 * (i >> 3) + 8 * j4 + (i & 4)];
        if (live) qmax = fmaxf(qmax, fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w))));
    }
    qmax = fmaxf(qmax, __shfl_xor(qmax, 16));
    qmax = fmaxf(qmax, __shfl_xor(qmax, 32));
    const int eq = query_exponent(qmax);
    const float qdown = u2f((uint32_t)(127 - eq) << 23);
    half8_t qh[NG], ql[NG];
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            const float4 f = *(const float4*)&smem[l16 * D + 32 * g + 8 * j4 + e];
            const float x[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                _Float16 hi, lo;
                split_hilo(live ? x[i] * qdown : 0.0f, hi, lo);
                qh[g][e + i] = hi;
                ql[g][e + i] = lo;
            }
        }
    __syncthreads();   // every wave has its query: the space is free
    float* ksl = smem + wave * OW;
    float* vsl = ksl + 256 * SCL;
    const float sscale = score_scale(D, eq);
    // the last cache row that the lane's column sees, and the tile's first and last column
    const int first_last = jb.past + col0 / p.group, last_last = jb.past + (col0 + gt - 1) / p.group;
    const int my_last = live ? jb.past + (col0 + l16) / p.group : last_last;
    const bool store = p.score_cols > 0 && live && col0 + l16 >= jb.count0 * p.group;
    float* score_at = (float*)(ws + p.scores) +
                      (((size_t)jb.page0 + (size_t)w.head * page_room(w.pages)) * p.score_cols + l16) * 64 + 4 * j4;
    const size_t pstride = (size_t)c.nKV * c.blk, hoff = (size_t)w.head * c.blk;
    auto page_rsrc = [&](const uint8_t* pool, int i) {
        const uint32_t pg = __builtin_amdgcn_readlane(pgv, i);
        const bool ok = pg < (uint32_t)c.n_pages;   // an index outside the cache: the page reads as zero, and is masked
        return __builtin_amdgcn_make_buffer_rsrc((void*)(pool + (ok ? (size_t)pg * pstride + hoff : 0)), 0,
                                                 ok ? c.blk : 0, 0x00020000);
    };
    const int vk = l16 * D + (D / 4) * j4, vv = j4 * D * 16 + l16 * 16;
    int vso[SCL];
#pragma unroll
    for (int s = 0; s < SCL; s++) {
        const int e = 256 * s + lane * 4, b = e >> 6, jb4 = (e >> 4) & 3;
        vso[s] = e < 64 * NG ? 4 * ((jb4 * NG + b) * 16 + (e & 15)) : c.blk;   // D = 64: the upper lanes read zero
    }
    float M = -INFINITY, lsum = 0.0f;
    // lane 16 j + .., entry s: of group 4 s + j, whose O is relative to 2^ev; the largest ev yet
    int ev[SCL], etop[SCL];
#pragma unroll
    for (int s = 0; s < SCL; s++) ev[s] = etop[s] = -127;
    float4_t o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] = float4_t{0.f, 0.f, 0.f, 0.f};
    u32x4 kc[4][NG / 2], vc[DT], kst[SCL], vst[SCL];
    auto load_k = [&](__amdgpu_buffer_rsrc_t rk, __amdgpu_buffer_rsrc_t rv) {
#pragma unroll
        for (int s = 0; s < SCL; s++) {
            kst[s] = __builtin_amdgcn_raw_buffer_load_b128(rk, lane * 16, 64 * D + 1024 * s, 0);
            vst[s] = __builtin_amdgcn_raw_buffer_load_b128(rv, vso[s], 64 * D, 0);
        }
#pragma unroll
        for (int tt = 0; tt < 4; tt++)
#pragma unroll
            for (int s = 0; s < NG / 2; s++)
                kc[tt][s] = __builtin_amdgcn_raw_buffer_load_b128(rk, vk, tt * 16 * D + 16 * s, 0);
    };
    auto load_v = [&](__amdgpu_buffer_rsrc_t rv) {
#pragma unroll
        for (int dt = 0; dt < DT; dt++) vc[dt] = __builtin_amdgcn_raw_buffer_load_b128(rv, vv, dt * 256, 0);
    };
    auto page = [&](int i) {
        const int in = i + 1 < nw ? i + 1 : i;
        const int p64 = 64 * (w0 + i);
        const bool bad = (uint32_t)__builtin_amdgcn_readlane(pgv, i) >= (uint32_t)c.n_pages;
        const int last = bad ? -1 : my_last;                // the last row that counts for the lane's column
        const int any_last = bad ? -1 : last_last;          // .. for one of them
        const bool edge = bad || p64 + 63 > first_last;     // a row that not every column sees
        int by[SCL];   // what brings O from the page before to this one's exponent
#pragma unroll
        for (int s = 0; s < SCL; s++) {
            *(u32x4*)&ksl[256 * s + lane * 4] = kst[s];
            if (edge) {   // rows past the tile's: whatever scale lies there, NaN too, goes in as zero
                const int t0 = p64 + 16 * (lane & 3) + 4 * (((256 * s + lane * 4) >> 4) & 3);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (t0 + e > any_last) vst[s][e] = 0u;
            }
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) top = max(top, finite_bits(vst[s][e]));
            const uint32_t mx = row_max_u32(top);
            const int en = max(mx ? min((int)(mx >> 23) - 127, 127) : ev[s], etop[s] - 60);
            etop[s] = max(etop[s], en);
            by[s] = ev[s] - en;
            ev[s] = en;
            const float down = u2f((uint32_t)(en < 127 ? 127 - en : 1) << 23) * (en < 127 ? 1.0f : 0.5f);   // 2^-en
            u32x4 v;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = f2u(u2f(vst[s][e]) * down);
            *(u32x4*)&vsl[256 * s + lane * 4] = v;
        }
        float pr[4][4];
        float pm = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < 4; tt++) {
            float ks[4 * NG];
#pragma unroll
            for (int s = 0; s < NG; s++) {
                const float4 f = *(const float4*)&ksl[(tt * 16 + 4 * j4) * NG + 4 * s];
                ks[4 * s] = f.x; ks[4 * s + 1] = f.y; ks[4 * s + 2] = f.z; ks[4 * s + 3] = f.w;
            }
            float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const u32x4 kw = kc[tt][g >> 1];
                const half8_t kf = (g & 1) ? dequant8_biased(kw[2], kw[3]) : dequant8_biased(kw[0], kw[1]);
                float4_t pp = {0.f, 0.f, 0.f, 0.f};
                pp = mfma16x16x32(kf, qh[g], pp);
                pp = mfma16x16x32(kf, ql[g], pp);
#pragma unroll
                for (int r = 0; r < 4; r++) acc[r] = __builtin_fmaf(ks[r * NG + g], pp[r], acc[r]);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) pr[tt][r] = acc[r];
        }
        if (edge) {
#pragma unroll
            for (int tt = 0; tt < 4; tt++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (p64 + tt * 16 + 4 * j4 + r > last) pr[tt][r] = -INFINITY;
        }
        if (store) {
#pragma unroll
            for (int tt = 0; tt < 4; tt++)
                *(float4_t*)(score_at + (size_t)(w0 + i) * p.score_cols * 64 + 16 * tt) =
                    float4_t{pr[tt][0], pr[tt][1], pr[tt][2], pr[tt][3]} * sscale;
        }
#pragma unroll
        for (int tt = 0; tt < 4; tt++)
#pragma unroll
            for (int r = 0; r < 4; r++) pm = fmaxf(pm, pr[tt][r]);
        const auto rvn = page_rsrc(c.v, in);
        load_k(page_rsrc(c.k, in), rvn);
        __builtin_amdgcn_sched_barrier(0);
        pm = fmaxf(pm, __shfl_xor(pm, 16));
        pm = fmaxf(pm, __shfl_xor(pm, 32));
        const float Mn = fmaxf(M, ceilf(pm * sscale));
        const float alpha = pow2_diff(M, Mn);
        lsum *= alpha;
#pragma unroll
        for (int b = 0; b < NG; b++) {
            const float alpha_o = ldexpf(alpha, __builtin_amdgcn_readlane(by[b >> 2], 16 * (b & 3)));
#pragma unroll
            for (int r = 0; r < 4; r++) {
                o[2 * b][r] *= alpha_o;
                o[2 * b + 1][r] *= alpha_o;
            }
        }
        const float base = P_SHIFT - (Mn == -INFINITY ? 0.0f : Mn);
        const bool large = __any(!(fabsf(base) < M_LARGE));
#pragma unroll
        for (int tt = 0; tt < 4; tt++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float t = __builtin_fmaf(pr[tt][r], sscale, base);
                if (large) t = pr[tt][r] * sscale - (Mn == -INFINITY ? 0.0f : Mn) + P_SHIFT;
                const float e = __builtin_amdgcn_exp2f(t);
                pr[tt][r] = e;
                lsum += e;
            }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < NG; b++) {
            float sv[16];
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const float4 f = *(const float4*)&vsl[b * 64 + 16 * j4 + 4 * s];
                sv[4 * s] = f.x; sv[4 * s + 1] = f.y; sv[4 * s + 2] = f.z; sv[4 * s + 3] = f.w;
            }
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
                u32x4 phw, plw;
#pragma unroll
                for (int ii = 0; ii < 8; ii += 2) {
                    const int tt = 2 * ks + (ii >> 2), r = ii & 3;
                    float x0 = pr[tt][r] * sv[4 * tt + r], x1 = pr[tt][r + 1] * sv[4 * tt + r + 1];
                    if (edge) {   // a row that this column does not see, whose scale is no finite number
                        if (p64 + tt * 16 + 4 * j4 + r > last) x0 = 0.0f;
                        if (p64 + tt * 16 + 4 * j4 + r + 1 > last) x1 = 0.0f;
                    }
                    uint32_t h, l;
                    split_hilo2(x0, x1, h, l);
                    phw[ii >> 1] = h;
                    plw[ii >> 1] = l;
                }
                const half8_t ph = __builtin_bit_cast(half8_t, phw), pl = __builtin_bit_cast(half8_t, plw);
#pragma unroll
                for (int dd = 0; dd < 2; dd++) {
                    const int dt = 2 * b + dd;
                    const u32x4 vw = vc[dt];
                    const half8_t vf = ks ? dequant8_biased(vw[2], vw[3]) : dequant8_biased(vw[0], vw[1]);
                    o[dt] = mfma16x16x32(vf, ph, o[dt]);
                    o[dt] = mfma16x16x32(vf, pl, o[dt]);
                }
            }
        }
        M = Mn;
        load_v(rvn);
    };
    if (nw > 0) {
        const auto rv = page_rsrc(c.v, 0);
        load_k(page_rsrc(c.k, 0), rv);
        load_v(rv);
        for (int i = 0; i < nw; i++) page(i);
    }
    lsum += __shfl_xor(lsum, 16);
    lsum += __shfl_xor(lsum, 32);
    {
        float* part = smem + wave * OW;   // its scale slices are this wave's own and done with
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
            *(float4_t*)(part + l16 * D + dt * 16 + 4 * j4) =
                o[dt] * ldexpf(P_UNSHIFT, __builtin_amdgcn_readlane(ev[dt >> 3], 16 * ((dt >> 1) & 3)));
        if (j4 == 0) {
            part[16 * D + l16] = M;
            part[16 * D + 16 + l16] = lsum * P_UNSHIFT;
        }
    }
    __syncthreads();
    // the four waves' parts, two channels a thread
    const size_t unit = (size_t)jb.unit0 + ((size_t)w.head * w.tiles + w.tile) * w.splits + w.split;
    float* mine = (float*)(ws + p.parts) + unit * 16 * D;
    float2* ml = (float2*)(ws + p.ml) + unit * 16;
    for (int i = tid; i < gt * (D / 2); i += 256) {
        const int h = i / (D / 2), d = 2 * (i & (D / 2 - 1));
        float m = -INFINITY;
#pragma unroll
        for (int v = 0; v < 4; v++) m = fmaxf(m, smem[v * OW + 16 * D + h]);
        float l = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const float* part = smem + v * OW;
            const float f = pow2_diff(part[16 * D + h], m);
            const float2 xy = *(const float2*)(part + h * D + d);
            l = __builtin_fmaf(part[16 * D + 16 + h], f, l);
            x = __builtin_fmaf(xy.x, f, x);
            y = __builtin_fmaf(xy.y, f, y);
        }
        if (w.splits == 1) {
            const int col = col0 + h;
            float* dst = out + ((int64_t)jb.row0 + col / p.group) * ldo + (size_t)(w.head * p.group + col % p.group) * D + d;
            dst[0] = l != 0.0f ? x / l : 0.0f;
            dst[1] = l != 0.0f ? y / l : 0.0f;
        } else {
            *(float2*)(mine + (size_t)h * D + d) = make_float2(x, y);
        }
        if (d == 0) ml[h] = make_float2(m, l);
    }
}

// M and 1/l of a column over its unit's splits (0 where it sees nothing), the
// splits' sums in their order; at: the first split's (M, l), `stride` from one
// split to the next.
__device__ static inline float2 column_total(const float2* __restrict__ at, int splits, int stride) {
    float m = -INFINITY, l = 0.0f;
    for (int s = 0; s < splits; s++) {
        const float2 v = at[(size_t)s * stride];
        const float mn = fmaxf(m, v.x);
        l = l * pow2_diff(m, mn) + v.y * pow2_diff(v.x, mn);
        m = mn;
    }
    return make_float2(m, l != 0.0f ? 1.0f / l : 0.0f);
}

// After k_weigh: joins the splits' outputs (the first jobs.joins workgroups,
// WEIGH_JOIN floats of a 16-column piece each, its splits dealt to four waves),
// and, from the stored scores, adds up the weights of FINISH_PAGES pages of a
// (job, kv head) a workgroup, a token a lane.
template <int NG>
__global__ __launch_bounds__(256) void k_weigh_finish(CacheDev c, WeighJobs jobs, WeighPlan p, MarksDev marks,
                                                      float* __restrict__ out, int64_t ldo, const uint8_t* __restrict__ ws) {
    constexpr int D = 32 * NG, CH = 16 * D / WEIGH_JOIN;   // chunks of a 16-column piece
    __shared__ __align__(16) float red[4][WEIGH_JOIN];
    __shared__ float2 total[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float2* ml = (const float2*)(ws + p.ml);
    if ((int)blockIdx.x < jobs.joins * CH) {
        const int piece = (int)blockIdx.x / CH, ch = (int)blockIdx.x % CH;
        const WeighJob jb = jobs.j[weigh_job_at(jobs, piece, &WeighJob::join0)];
        const int tiles = weigh_tiles(jb, p), splits = (weigh_pages(jb) + p.per - 1) / p.per;
        if (splits == 1) return;   // the attention kernel wrote them
        const int r = piece - jb.join0, sub = r % p.subs, tile = r / p.subs % tiles, head = r / p.subs / tiles;
        const int col0 = (tile * p.subs + sub) * 16, gt = min(16, jb.n * p.group - col0);
        const int h = (ch * WEIGH_JOIN + lane * 4) / D, d = (ch * WEIGH_JOIN + lane * 4) % D;
        if (ch * WEIGH_JOIN / D >= gt) return;
        const size_t unit = (size_t)jb.unit0 + ((size_t)head * tiles + tile) * splits;
        const float2* at = ml + (unit * p.subs + sub) * 16 + h;
        const float* part = (const float*)(ws + p.parts) + (unit * p.subs + sub) * 16 * D + ch * WEIGH_JOIN + lane * 4;
        float m = -INFINITY, l = 0.0f;
        float4_t x = {0.f, 0.f, 0.f, 0.f};
        if (h < gt) {
#pragma unroll 4
            for (int s = wave; s < splits; s += 4) {
                const float2 v = at[(size_t)s * p.subs * 16];
                const float4_t y = *(const float4_t*)(part + (size_t)s * p.subs * 16 * D);
                const float mn = fmaxf(m, v.x), fa = pow2_diff(m, mn), fb = pow2_diff(v.x, mn);
                l = l * fa + v.y * fb;
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = x[e] * fa + y[e] * fb;
                m = mn;
            }
        }
        __shared__ float2 wml[4][64];
        wml[wave][lane] = make_float2(m, l);
        *(float4_t*)&red[wave][lane * 4] = x;
        __syncthreads();
        if (wave || h >= gt) return;
        for (int v = 1; v < 4; v++) {
            const float2 o = wml[v][lane];
            const float4_t y = *(const float4_t*)&red[v][lane * 4];
            const float mn = fmaxf(m, o.x), fa = pow2_diff(m, mn), fb = pow2_diff(o.x, mn);
            l = l * fa + o.y * fb;
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = x[e] * fa + y[e] * fb;
            m = mn;
        }
        const int col = col0 + h;
        float* dst = out + ((int64_t)jb.row0 + col / p.group) * ldo + (size_t)(head * p.group + col % p.group) * D + d;
#pragma unroll
        for (int e = 0; e < 4; e++) dst[e] = l != 0.0f ? x[e] / l : 0.0f;
        return;
    }
    const int u = ((int)blockIdx.x - jobs.joins * CH) * FINISH_PAGES;
    const WeighJob jb = jobs.j[weigh_job_at(jobs, u, &WeighJob::page0)];
    const int pages = weigh_pages(jb), room = page_room(pages);
    const int head = (u - jb.page0) / room, p0 = (u - jb.page0) % room;
    const int splits = (pages + p.per - 1) / p.per;
    const int c0 = jb.count0 * p.group, cols = jb.n * p.group;
    const size_t unit = (size_t)jb.unit0 + (size_t)head * splits;
    if (tid < cols) total[tid] = column_total(ml + unit * 16 + tid, splits, 16);
    __syncthreads();
    for (int i = wave; i < FINISH_PAGES && p0 + i < pages; i += 4) {
        const int pg = p0 + i;
        const uint32_t id = c.page_table[(size_t)jb.slot * c.max_pages + pg];
        if (id >= (uint32_t)c.n_pages || 64 * pg + lane >= jb.past + jb.n) continue;
        float* wt = marks.weight + ((size_t)id * c.nKV + head) * 64 + lane;
        const float* s = (const float*)(ws + p.scores) + ((size_t)jb.page0 + (size_t)head * room + pg) * p.score_cols * 64 + lane;
        const float before = p.fade == 0.0f && 64 * pg + lane >= jb.fresh ? 0.0f : *wt;
        float got = 0.0f;
        for (int col = c0; col < cols; col++) {
            const float2 t = total[col];
            const float x = __builtin_amdgcn_exp2f(s[(size_t)col * 64] - (t.x == -INFINITY ? 0.0f : t.x));
            got = __builtin_fmaf(x, t.y, got);
        }
        *wt = __builtin_fmaf(before, 64 * pg + lane >= jb.fresh ? p.fade : 1.0f, got);
    }
}

// The queries of many columns, rotated once, as the matrix products take them:
// a piece of 16 columns is [hi, lo][NG][64 lanes] of 8 f16, and its scale for
// the scores 16 f32.
template <int NG>
__global__ __launch_bounds__(256) void k_weigh_query(CacheDev c, WeighJobs jobs, WeighPlan p, AxesDev axes,
                                                     const float* __restrict__ q, int64_t ldq, uint8_t* __restrict__ ws) {
    constexpr int D = 32 * NG;
    __shared__ __align__(16) float x[16 * D];
    __shared__ int s_eq[16];
    const int tid = threadIdx.x, piece = blockIdx.x;
    const WeighJob jb = jobs.j[weigh_job_at(jobs, piece, &WeighJob::join0)];
    const int per_head = weigh_tiles(jb, p) * p.subs, r = piece - jb.join0, head = r / per_head;
    const int col0 = r % per_head * 16, gt = max(0, min(16, jb.n * p.group - col0));
    for (int i = tid; i < 16 * (D / 8); i += 256) {
        const int h = i / (D / 8), d0 = 8 * (i & (D / 8 - 1));
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (h < gt) query8(c, axes, jb, p, head, col0 + h, d0, q, ldq, v);
        *(float4*)&x[h * D + d0] = make_float4(v[0], v[1], v[2], v[3]);
        *(float4*)&x[h * D + d0 + 4] = make_float4(v[4], v[5], v[6], v[7]);
    }
    __syncthreads();
    {   // 16 threads a column
        float m = 0.0f;
        for (int d = tid & 15; d < D; d += 16) m = fmaxf(m, fabsf(x[(tid >> 4) * D + d]));
        for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
        if ((tid & 15) == 0) {
            s_eq[tid >> 4] = query_exponent(m);
            ((float*)(ws + p.qs))[(size_t)piece * 16 + (tid >> 4)] = score_scale(D, query_exponent(m));
        }
    }
    __syncthreads();
    u32x4* to = (u32x4*)(ws + p.q) + (size_t)piece * 2 * NG * 64;
    for (int i = tid; i < NG * 64; i += 256) {
        const int lane = i & 63, g = i >> 6, h = lane & 15;
        const float down = u2f((uint32_t)(127 - s_eq[h]) << 23);
        half8_t hi, lo;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            _Float16 a, b;
            split_hilo(x[h * D + 32 * g + 8 * (lane >> 4) + e] * down, a, b);
            hi[e] = a;
            lo[e] = b;
        }
        to[i] = __builtin_bit_cast(u32x4, hi);
        to[NG * 64 + i] = __builtin_bit_cast(u32x4, lo);
    }
}

// 8 codes times a scale, in 2^7 .. 2^15 where they are largest, as an f16 pair.
__device__ static inline void code_pair(uint32_t lo4, uint32_t hi4, float scale, half8_t& hi, half8_t& lo) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float x = (float)((int)(((e < 4 ? lo4 : hi4) >> (8 * (e & 3))) & 0xffu) - 128) * scale;
        _Float16 a, b;
        split_hilo(x, a, b);
        hi[e] = a;
        lo[e] = b;
    }
}
// The exponent of the largest of a page's scales (bits), within what the pair's
// scale can be: 2^-pair_down(e) brings a scale to 2^7 .. 2^8.
__device__ static inline int pair_exponent(uint32_t top) { return max((int)(top >> 23) - 127, -112); }
__device__ static inline float pair_down(int e) { return u2f((uint32_t)(134 - e) << 23); }

// The weights from many columns: q . k again, with the columns' M and l known.
// A wave holds the keys of 16 * TT rows of the cache as f16 pairs in registers
// and walks the columns, 16 at a time; a lane adds up its 4 * TT rows' p / l,
// and 16 lanes meet at the end, in a fixed order.
template <int NG>
__global__ __launch_bounds__(256, 2) void k_weigh_sums(CacheDev c, WeighJobs jobs, WeighPlan p, MarksDev marks,
                                                       const uint8_t* __restrict__ ws) {
    constexpr int D = 32 * NG, TT = NG > 4 ? 2 : 4, PER_PAGE = 4 / TT;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, j4 = lane >> 4, l16 = lane & 15;
    constexpr int WGS = FINISH_PAGES * PER_PAGE / 4;   // workgroups of FINISH_PAGES pages
    const int u = (int)blockIdx.x / WGS * FINISH_PAGES;
    const WeighJob jb = jobs.j[weigh_job_at(jobs, u, &WeighJob::page0)];
    if (jb.count0 >= jb.n) return;   // a piece of a job before the rows that count
    const int pages = weigh_pages(jb), room = page_room(pages), head = (u - jb.page0) / room;
    const int part = (u - jb.page0) % room * PER_PAGE + (int)blockIdx.x % WGS * 4 + wave;   // 16 * TT rows each
    const int pg = part / PER_PAGE, r0 = part * 16 * TT;     // the first of the wave's rows
    if (pg >= pages) return;
    const uint32_t id = c.page_table[(size_t)jb.slot * c.max_pages + pg];
    if (id >= (uint32_t)c.n_pages) return;
    const int held = jb.past + jb.n;
    const uint8_t* blk = c.k + ((size_t)id * c.nKV + head) * c.blk;
    half8_t kh[TT][NG], kl[TT][NG];
    int e;
    {
        float sc[TT][NG];
        uint32_t top = 0;
#pragma unroll
        for (int tt = 0; tt < TT; tt++) {
            const int r = r0 + 16 * tt + l16;
            const float* at = (const float*)(blk + 64 * D) + (r & 63) * NG;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                sc[tt][g] = r < held ? at[g] : 0.0f;
                top = max(top, finite_bits(f2u(sc[tt][g])));
            }
        }
        e = pair_exponent(row_max_u32(top));
        const float down = pair_down(e);
#pragma unroll
        for (int tt = 0; tt < TT; tt++)
#pragma unroll
            for (int g = 0; g < NG; g += 2) {
                const u32x4 w = *(const u32x4*)(blk + (size_t)((r0 & 63) + 16 * tt + l16) * D + (D / 4) * j4 + 8 * g);
                code_pair(w[0], w[1], sc[tt][g] * down, kh[tt][g], kl[tt][g]);
                code_pair(w[2], w[3], sc[tt][g + 1] * down, kh[tt][g + 1], kl[tt][g + 1]);
            }
    }
    const int splits = (pages + p.per - 1) / p.per, tiles = weigh_tiles(jb, p);
    const int c0 = jb.count0 * p.group, cols = jb.n * p.group;
    const int from = max(c0, max(0, r0 - jb.past) * p.group);   // the first column that sees one of the wave's rows
    float4_t got[TT];
#pragma unroll
    for (int tt = 0; tt < TT; tt++) got[tt] = float4_t{0.f, 0.f, 0.f, 0.f};
    for (int t16 = from / 16; t16 * 16 < cols; t16++) {
        const size_t piece = (size_t)jb.join0 + (size_t)head * tiles * p.subs + t16;
        const u32x4* qf = (const u32x4*)(ws + p.q) + piece * 2 * NG * 64 + lane;
        float4_t acc[TT];
#pragma unroll
        for (int tt = 0; tt < TT; tt++) acc[tt] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const half8_t qh = __builtin_bit_cast(half8_t, qf[g * 64]), ql = __builtin_bit_cast(half8_t, qf[(NG + g) * 64]);
#pragma unroll
            for (int tt = 0; tt < TT; tt++) {
                acc[tt] = mfma16x16x32(kh[tt][g], qh, acc[tt]);
                acc[tt] = mfma16x16x32(kl[tt][g], qh, acc[tt]);
                acc[tt] = mfma16x16x32(kh[tt][g], ql, acc[tt]);
            }
        }
        const int col = t16 * 16 + l16;
        const float2 t = column_total((const float2*)(ws + p.ml) +
                                          (((size_t)jb.unit0 + ((size_t)head * tiles + t16 / p.subs) * splits) * p.subs + t16 % p.subs) * 16 + l16,
                                      splits, p.subs * 16);
        const float sc = ldexpf(((const float*)(ws + p.qs))[piece * 16 + l16], e - 7);
        const float base = t.x == -INFINITY ? 0.0f : -t.x;
        const bool large = __any(!(fabsf(base) < M_LARGE));
        const int last = col >= c0 && col < cols ? jb.past + col / p.group : -1;
        const bool edge = t16 * 16 < c0 || t16 * 16 + 16 > cols || jb.past + t16 * 16 / p.group < r0 + 16 * TT - 1;
#pragma unroll
        for (int tt = 0; tt < TT; tt++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float a = __builtin_fmaf(acc[tt][r], sc, base);
                if (large && a > 0.0f) a = 0.0f;   // its rounding alone can be above M
                const float x = __builtin_amdgcn_exp2f(a) * t.y;
                got[tt][r] += edge && r0 + 16 * tt + 4 * j4 + r > last ? 0.0f : x;
            }
    }
#pragma unroll
    for (int tt = 0; tt < TT; tt++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            for (int o = 1; o < 16; o <<= 1) got[tt][r] += __shfl_xor(got[tt][r], o);
    if (l16) return;
    float* wt = marks.weight + ((size_t)id * c.nKV + head) * 64;
#pragma unroll
    for (int tt = 0; tt < TT; tt++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int row = r0 + 16 * tt + 4 * j4 + r;
            if (row >= held) continue;
            const bool fades = row >= jb.fresh;
            const float before = fades && p.fade == 0.0f ? 0.0f : wt[row & 63];
            wt[row & 63] = __builtin_fmaf(before, fades ? p.fade : 1.0f, got[tt][r]);
        }
}

template <int NG>
static hipError_t weigh_ng(hipStream_t st, const CacheDev& c, const WeighJobs& jobs, const WeighPlan& p, bool few,
                           const AxesDev& axes, const MarksDev& marks, const float* q, int64_t ldq, float* out, int64_t ldo,
                           uint8_t* ws) {
    constexpr int D = 32 * NG, CH = 16 * D / WEIGH_JOIN, PER_PAGE = NG > 4 ? 2 : 1;
    hipError_t e = hipSuccess;
    if (!few && p.weigh) e = op_launch(k_weigh_query<NG>, dim3(jobs.joins), dim3(256), st, c, jobs, p, axes, q, ldq, ws);
    if (e == hipSuccess)
        e = op_launch(k_weigh<NG>, dim3(op_blocks(jobs.units)), dim3(256), st, c, jobs, p, axes, q, ldq, out, ldo, ws);
    bool split = false;
    for (int j = 0; j < jobs.n; j++) split = split || weigh_pages(jobs.j[j]) > p.per;
    WeighJobs finish = jobs;
    if (!split) finish.joins = 0;
    const int blocks = finish.joins * CH + (few && p.weigh ? jobs.pages / FINISH_PAGES : 0);
    if (e == hipSuccess && blocks)
        e = op_launch(k_weigh_finish<NG>, dim3(blocks), dim3(256), st, c, finish, p, marks, out, ldo, ws);
    if (e == hipSuccess && !few && p.weigh)
        e = op_launch(k_weigh_sums<NG>, dim3(jobs.pages * PER_PAGE / 4), dim3(256), st, c, jobs, p, marks, ws);
    return e;
}

hipError_t launch_weigh(hipStream_t st, const CacheDev& c, const WeighJobs& jobs, const WeighPlan& plan, bool few,
                        const AxesDev& axes, const MarksDev& marks, const float* q, int64_t ldq, float* out, int64_t ldo,
                        uint8_t* ws) {
    WeighPlan p = plan;
    p.vec = aligned16(q) && aligned16(c.rope) && ldq % 4 == 0 && c.rot % 16 == 0;
    if (c.ng == 2) return weigh_ng<2>(st, c, jobs, p, few, axes, marks, q, ldq, out, ldo, ws);
    if (c.ng == 4) return weigh_ng<4>(st, c, jobs, p, few, axes, marks, q, ldq, out, ldo, ws);
    return weigh_ng<8>(st, c, jobs, p, few, axes, marks, q, ldq, out, ldo, ws);
}

// ================================================================== evict ===
// What a row is kept by: its weight's order-preserving bits (-0 as 0; one that
// is no number counts least), above every weight where its token is one of the
// chat's first or latest.
__device__ static inline uint32_t keep_key(float weight, int token, int sink, int latest) {
    if (token < sink || token >= latest) return 0xffffffffu;
    return weight != weight ? 0u : order_bits(weight + 0.0f);
}

// One row's codes, scales and marks to another row of the same slot and kv
// head, by a wave.
template <int NG>
__device__ static inline void move_row(const CacheDev& c, const MarksDev& marks, const uint32_t* pt, int head, int of, int to,
                                       int lane) {
    constexpr int D = 32 * NG;
    const uint32_t pf = pt[of >> 6], ptt = pt[to >> 6];
    if (pf >= (uint32_t)c.n_pages || ptt >= (uint32_t)c.n_pages) return;
    const size_t bf = (size_t)pf * c.nKV + head, bt = (size_t)ptt * c.nKV + head;
    const int s = of & 63, t = to & 63;
    const uint8_t *kf = c.k + bf * c.blk, *vf = c.v + bf * c.blk;
    uint8_t *kt = c.k + bt * c.blk, *vt = c.v + bt * c.blk;
    if (lane < D / 4) *(uint32_t*)(kt + t * D + 4 * lane) = *(const uint32_t*)(kf + s * D + 4 * lane);
#pragma unroll
    for (int i = 0; i < D / 64; i++) vt[vcode_at(lane + 64 * i, t, D)] = vf[vcode_at(lane + 64 * i, s, D)];
    if (lane < NG) {
        *(uint32_t*)(kt + 64 * D + 4 * (t * NG + lane)) = *(const uint32_t*)(kf + 64 * D + 4 * (s * NG + lane));
        *(uint32_t*)(vt + 64 * D + 4 * vscale_at(lane, t, NG)) = *(const uint32_t*)(vf + 64 * D + 4 * vscale_at(lane, s, NG));
    }
    if (lane == 32) marks.weight[bt * 64 + t] = marks.weight[bf * 64 + s];
    if (lane == 33) marks.token[bt * 64 + t] = marks.token[bf * 64 + s];
}

// A workgroup of 1024 finds the rows that one (job, kv head) keeps. A thread
// holds a run of rows' keys (REG of them in registers; 0: as many as it takes,
// read again for each pass); the keep-th largest key comes from three passes
// over 11, 11 and 10 bits from the top with a histogram in LDS, and of its
// equals the lower rows stay. The rows below `keep` that go and the rows from
// `keep` on that stay are as many, and the i-th of the one takes the place of
// the i-th of the other: `of` and `to` lists in the workspace, or up to
// EVICT_HERE moves made here.
template <int NG, int REG>
__global__ __launch_bounds__(1024) void k_evict_select(CacheDev c, EvictJobs jobs, MarksDev marks, int sink, int recent,
                                                       uint8_t* __restrict__ ws) {
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t wsum[2][16];
    __shared__ uint32_t s_sel[2];
    __shared__ int here_of[EVICT_HERE], here_to[EVICT_HERE];
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
#pragma unroll
        for (int e = 0; e < REG; e += 4) {
            float4 w = {0.f, 0.f, 0.f, 0.f};
            int4 k = {0, 0, 0, 0};
            if (ok) {
                w = *(const float4*)(marks.weight + m + e);
                k = *(const int4*)(marks.token + m + e);
            }
            reg[e] = ok ? keep_key(w.x, k.x, sink, latest) : 0u;
            reg[e + 1] = ok ? keep_key(w.y, k.y, sink, latest) : 0u;
            reg[e + 2] = ok ? keep_key(w.z, k.z, sink, latest) : 0u;
            reg[e + 3] = ok ? keep_key(w.w, k.w, sink, latest) : 0u;
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
    // what the threads before this one have of a and b
    auto before = [&](uint32_t& a, uint32_t& b) {
        uint32_t x = a, y = b;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t u = __shfl_up(x, o), v = __shfl_up(y, o);
            if (lane >= o) {
                x += u;
                y += v;
            }
        }
        if (lane == 63) {
            wsum[0][wave] = x;
            wsum[1][wave] = y;
        }
        __syncthreads();
        x -= a;
        y -= b;
        for (int w = 0; w < wave; w++) {
            x += wsum[0][w];
            y += wsum[1][w];
        }
        __syncthreads();
        a = x;
        b = y;
    };
    uint32_t prefix = 0, left = (uint32_t)jb.keep;
#pragma unroll
    for (int ps = 0; ps < 3; ps++) {
        const int sh = ps == 0 ? 21 : ps == 1 ? 10 : 0, bits = ps == 2 ? 10 : 11;
        const uint32_t mask = (1u << bits) - 1;
        hist[t] = hist[t + 1024] = 0;
        __syncthreads();
        each([&](int, uint32_t k) {
            if (ps == 0 || k >> (sh + bits) % 32 == prefix >> (sh + bits) % 32) atomicAdd(&hist[(k >> sh) & mask], 1u);
        });
        __syncthreads();
        // thread t: the digits 2047 - 2t and 2046 - 2t, from the largest down
        const uint32_t n0 = hist[2047 - 2 * t], n1 = hist[2046 - 2 * t];
        uint32_t b0 = n0 + n1, none = 0;
        before(b0, none);
        if (b0 < left && left <= b0 + n0 + n1) {
            const bool first = left <= b0 + n0;
            s_sel[0] = prefix | (uint32_t)(2047 - 2 * t - (first ? 0 : 1)) << sh;
            s_sel[1] = left - b0 - (first ? 0 : n0);
        }
        __syncthreads();
        prefix = s_sel[0];
        left = s_sel[1];
    }
    // prefix: the keep-th largest key; `left` of the rows that have it stay
    uint32_t eq = 0, none = 0;
    each([&](int, uint32_t k) { eq += k == prefix; });
    before(eq, none);
    uint32_t to = 0, of = 0, be = eq;
    auto kept = [&](uint32_t k) {
        const bool same = k == prefix, in = k > prefix || (same && be < left);
        be += same;
        return in;
    };
    each([&](int i, uint32_t k) {
        const bool in = kept(k);
        to += i < jb.keep && !in;
        of += i >= jb.keep && in;
    });
    const uint32_t mine = of;
    before(to, of);
    be = eq;
    const bool here = jb.room <= EVICT_HERE;
    int32_t* list = (int32_t*)ws + jb.moves0 + (int64_t)head * (2 * jb.room + 2);   // count, -, (of, to) pairs
    if (t == 1023) {
        const uint32_t n = min(of + mine, (uint32_t)jb.room);
        if (here) s_sel[0] = n;
        else list[0] = (int32_t)n;
    }
    each([&](int i, uint32_t k) {
        const bool in = kept(k);
        if (i < jb.keep && !in) {   // (within `room` unless another stream writes the marks meanwhile)
            if (here && to < EVICT_HERE) here_to[to] = i;
            if (!here && to < (uint32_t)jb.room) list[2 + 2 * to + 1] = i;
            to++;
        } else if (i >= jb.keep && in) {
            if (here && of < EVICT_HERE) here_of[of] = i;
            if (!here && of < (uint32_t)jb.room) list[2 + 2 * of] = i;
            of++;
        }
    });
    if (!here) return;
    __syncthreads();
    const int n = (int)s_sel[0];
    for (int i = wave; i < n; i += 16) move_row<NG>(c, marks, pt, head, here_of[i], here_to[i], lane);
}

// The moves of the lists: rows from `keep` on to rows below it, so no row is
// both read and written. A workgroup takes EVICT_MOVES of a (job, kv head)'s.
constexpr int EVICT_MOVES = 32;
template <int NG>
__global__ __launch_bounds__(256) void k_evict_move(CacheDev c, EvictJobs jobs, MarksDev marks,
                                                    const uint8_t* __restrict__ ws) {
    const EvictJob jb = jobs.j[blockIdx.y / c.nKV];
    const int head = (int)blockIdx.y % c.nKV, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (jb.room <= EVICT_HERE) return;
    const int32_t* list = (const int32_t*)ws + jb.moves0 + (int64_t)head * (2 * jb.room + 2);
    const int i0 = (int)blockIdx.x * EVICT_MOVES, n = min(list[0] - i0, EVICT_MOVES);
    const uint32_t* pt = c.page_table + (size_t)jb.slot * c.max_pages;
    for (int i = wave; i < n; i += 4) {
        const int2 m = *(const int2*)(list + 2 + 2 * (i0 + i));
        move_row<NG>(c, marks, pt, head, m.x, m.y, lane);
    }
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
        e = op_launch(k_evict_move<NG>, dim3((jobs.room + EVICT_MOVES - 1) / EVICT_MOVES, jobs.n * c.nKV), dim3(256), st, c,
                      jobs, marks, ws);
    return e;
}

hipError_t launch_evict(hipStream_t st, const CacheDev& c, const EvictJobs& jobs, int max_rows, const MarksDev& marks,
                        int sink, int recent, uint8_t* ws) {
    if (c.ng == 2) return evict_ng<2>(st, c, jobs, max_rows, marks, sink, recent, ws);
    if (c.ng == 4) return evict_ng<4>(st, c, jobs, max_rows, marks, sink, recent, ws);
    return evict_ng<8>(st, c, jobs, max_rows, marks, sink, recent, ws);
}
