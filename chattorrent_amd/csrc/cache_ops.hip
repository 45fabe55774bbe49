// Operators on a paged int8 cache in device memory (cc_cache): appending rows
// with the key bounds of the pages they complete, and attention over the pages
// that a cheap score selects. The cache is laid out as the pass lays its own
// out (common.h, KV geometry), so they run on a context's cache as well.
#include "common.h"
#include "ops.h"
#include <algorithm>

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));

// The job that holds unit u (uniform: u comes from the block's index).
__device__ static inline OpJob job_of(const OpJobs& jobs, int u) {
    int lo = 0, hi = jobs.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (jobs.j[mid].first <= u) lo = mid;
        else hi = mid;
    }
    return jobs.j[lo];
}

// ================================================================= append ===
// Rows of keys and values into their pages, and key bounds.
//
// A workgroup takes one (page that a job's rows touch, kv head, K or V). A
// lane holds 8 consecutive channels of a row, so D/8 lanes hold the row, a
// 32-channel group is 4 neighbouring lanes (its largest magnitude two
// exchanges away) and a wave takes 512/D rows at a time. RoPE, amax, scale =
// amax/127, inv = 1/scale, rint, clamp: the f32 steps of the pass's own store,
// so the codes and scales are its bits. 4000 rows of 8 heads of 128 (42 MB)
// take 15.5-16 us, 2.7 TB/s: half the rate of a copy. A wave of a whole page
// walks its strides of rows one after another, and loads the next when the one
// before is stored: a chain of four latencies. 32 rows take 4.4 us. Bounds
// alone, of 16 chats of 16384 tokens (311 MB): 160 us, 1.9 TB/s, the same walk.
//
// Key bounds (a page's, made when its 64th row is stored): per channel the
// largest and the smallest of the page's 64 dequantised keys, as codes against
// B = (largest magnitude in the 32-channel group)/127, the largest rounded up
// and the smallest down. Rows that were there before are read back from the
// page. Layout of a page's bounds: per kv head 2*D code bytes, channel d's
// largest (w = 0) or smallest (w = 1) at (2w + (d%32)/16)*(D/2) + 16*(d/32) +
// d%16, so that a lane of the score's matrix operand reads D/2 bytes in one
// run; then, after all kv heads' codes, B as f32 [kv heads][D/32].
__device__ static inline void bound_code(float mx, float mn, float B, int8_t& hi, int8_t& lo) {
    hi = lo = 0;
    if (!(B > 0.0f)) return;
    hi = (int8_t)(int)fminf(fmaxf(ceilf(mx / B), -127.0f), 127.0f);
    lo = (int8_t)(int)fminf(fmaxf(floorf(mn / B), -127.0f), 127.0f);
}

// Channels d0 .. d0 + 7 of one head of a row x, rotated with the position's
// (cos, sin) pairs cs: the f32 steps of rope_cs (rot 0: as they are). vec: x
// is 16-byte aligned at groups of 4 channels, as is cs, and RoPE's halves are
// whole groups of 8.
__device__ static inline void rotated8(const float* __restrict__ x, int d0, const float* __restrict__ cs, int rot,
                                       bool vec, float (&r)[8]) {
    const int half = rot >> 1;
    if (vec) {
        const float4 a = *(const float4*)(x + d0), b = *(const float4*)(x + d0 + 4);
        r[0] = a.x; r[1] = a.y; r[2] = a.z; r[3] = a.w;
        r[4] = b.x; r[5] = b.y; r[6] = b.z; r[7] = b.w;
        if (d0 < rot) {
            const bool low = d0 < half;
            const float* y = x + d0 + (low ? half : -half);
            const float4 ya = *(const float4*)y, yb = *(const float4*)(y + 4);
            const float o[8] = {ya.x, ya.y, ya.z, ya.w, yb.x, yb.y, yb.z, yb.w};
            const float4* t = (const float4*)(cs + 2 * (d0 - (low ? 0 : half)));
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float4 c = t[e >> 1];
                r[e] = low ? r[e] * c.x - o[e] * c.y : r[e] * c.x + o[e] * c.y;
                r[e + 1] = low ? r[e + 1] * c.z - o[e + 1] * c.w : r[e + 1] * c.z + o[e + 1] * c.w;
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int d = d0 + e;
        r[e] = x[d];
        if (d < rot) {
            const float* t = cs + 2 * (d < half ? d : d - half);
            const float o = x[d < half ? d + half : d - half];
            r[e] = d < half ? r[e] * t[0] - o * t[1] : r[e] * t[0] + o * t[1];
        }
    }
}

template <int D, bool VEC>
__global__ __launch_bounds__(256) void k_kv_append(CacheDev c, OpJobs jobs, const float* __restrict__ k, int64_t ldk,
                                                   const float* __restrict__ v, int64_t ldv, int only) {
    constexpr int G8 = D / 8, RPW = 64 / G8, NG = D / 32;
    __shared__ float red[2][4][D];
    const OpJob jb = job_of(jobs, blockIdx.x);
    const int head = blockIdx.y, which = blockIdx.z;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // bounds alone (`only`): the job's whole pages, each with 64 rows that were there before
    const int p = (jb.past + (only ? 63 : 0)) / 64 + ((int)blockIdx.x - jb.first);
    const int s0 = only ? 64 : max(jb.past - 64 * p, 0), s1 = only ? 64 : min(jb.past + jb.n - 64 * p, 64);
    const uint32_t page = c.page_table[(size_t)jb.slot * c.max_pages + p];
    if (page >= (uint32_t)c.n_pages) return;
    uint8_t* blk = (which ? c.v : c.k) + ((size_t)page * c.nKV + head) * c.blk;
    const int g = lane & (G8 - 1), rr = lane / G8;
    const bool bounds = which == 0 && c.bounds != nullptr && s1 == 64;
    float mx[8], mn[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        mx[e] = -INFINITY;
        mn[e] = INFINITY;
    }
    // rows that the page held before
    if (bounds)
        for (int s = wave * RPW + rr; s < s0; s += 4 * RPW) {
            const uint2 u = *(const uint2*)(blk + (size_t)s * D + kpos(8 * g, D));
            const float sc = *(const float*)(blk + 64 * D + ((size_t)s * NG + (g >> 2)) * 4);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int code = (int)(((e < 4 ? u.x : u.y) >> (8 * (e & 3))) & 0xffu) - 128;
                const float x = (float)code * sc;
                mx[e] = fmaxf(mx[e], x);
                mn[e] = fminf(mn[e], x);
            }
        }
    const float* src = (which ? v : k) + (size_t)head * D;
    const int64_t ld = which ? ldv : ldk;
    if (which == 1 && s1 - s0 == 64) {
        // a whole page of V: a thread takes 8 channels of 4 tokens in a row, whose codes of a channel lie beside each other,
        // and 4 neighbours in a wave (D <= 128) fill a channel's 16 bytes. (4000 rows of 8 x 128: 20 us with a byte a
        // store, 15.5 with these; two rows of K at a time: no better.)
        for (int i = threadIdx.x; i < 16 * G8; i += 256) {
            const int g8 = i & (G8 - 1), r = i / G8, t = 16 * (r & 3) + 4 * (r >> 2);   // tokens t .. t + 3
            uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            float sc[4];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                float x[8];
                rotated8(src + (jb.row0 + 64 * p + t + q - jb.past) * ld, 8 * g8, nullptr, 0, VEC, x);
                float amax = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(x[e]));
                amax = fmaxf(amax, __shfl_xor(amax, 1));
                amax = fmaxf(amax, __shfl_xor(amax, 2));
                sc[q] = amax / 127.0f;
                const float inv = sc[q] > 0.0f ? 1.0f / sc[q] : 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++)
                    w[e] |= (uint32_t)(((int)fminf(fmaxf(__builtin_rintf(x[e] * inv), -127.0f), 127.0f) ^ 0x80) & 0xff) << (8 * q);
            }
#pragma unroll
            for (int e = 0; e < 8; e++) *(uint32_t*)(blk + vcode_at(8 * g8 + e, t, D)) = w[e];
            if ((g8 & 3) == 0)
                *(float4*)(blk + 64 * D + (size_t)vscale_at(g8 >> 2, t, NG) * 4) = make_float4(sc[0], sc[1], sc[2], sc[3]);
        }
        return;
    }
    for (int sb = s0 + wave * RPW; sb < s1; sb += 4 * RPW) {   // uniform in the wave: lanes exchange below
        const int s = sb + rr;
        const bool live = s < s1;
        const int pos = 64 * p + (live ? s : s0);
        float r[8];
        rotated8(src + (jb.row0 + pos - jb.past) * ld, 8 * g, c.rope + (size_t)pos * c.rot, which == 0 ? c.rot : 0, VEC, r);
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(r[e]));
        amax = fmaxf(amax, __shfl_xor(amax, 1));
        amax = fmaxf(amax, __shfl_xor(amax, 2));
        const float scale = amax / 127.0f;
        const float inv = scale > 0.0f ? 1.0f / scale : 0.0f;
        if (!live) continue;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int code = (int)fminf(fmaxf(__builtin_rintf(r[e] * inv), -127.0f), 127.0f);
            w[e >> 2] |= (uint32_t)((code ^ 0x80) & 0xff) << (8 * (e & 3));
            const float x8 = (float)code * scale;
            mx[e] = fmaxf(mx[e], x8);
            mn[e] = fminf(mn[e], x8);
        }
        if (which == 0) {
            *(uint2*)(blk + (size_t)s * D + kpos(8 * g, D)) = make_uint2(w[0], w[1]);
            if ((g & 3) == 0) *(float*)(blk + 64 * D + ((size_t)s * NG + (g >> 2)) * 4) = scale;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) blk[vcode_at(8 * g + e, s, D)] = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
            if ((g & 3) == 0) *(float*)(blk + 64 * D + (size_t)vscale_at(g >> 2, s, NG) * 4) = scale;
        }
    }
    if (!bounds) return;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        for (int o = G8; o < 64; o <<= 1) {
            mx[e] = fmaxf(mx[e], __shfl_xor(mx[e], o));
            mn[e] = fminf(mn[e], __shfl_xor(mn[e], o));
        }
        if (rr == 0) {
            red[0][wave][8 * g + e] = mx[e];
            red[1][wave][8 * g + e] = mn[e];
        }
    }
    __syncthreads();
    if (threadIdx.x >= G8) return;
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int d = 8 * g + e;
        mx[e] = fmaxf(fmaxf(red[0][0][d], red[0][1][d]), fmaxf(red[0][2][d], red[0][3][d]));
        mn[e] = fminf(fminf(red[1][0][d], red[1][1][d]), fminf(red[1][2][d], red[1][3][d]));
        amax = fmaxf(amax, fmaxf(fabsf(mx[e]), fabsf(mn[e])));
    }
    amax = fmaxf(amax, __shfl_xor(amax, 1));
    amax = fmaxf(amax, __shfl_xor(amax, 2));
    const float B = amax / 127.0f;
    uint32_t w[2][2] = {{0, 0}, {0, 0}};
#pragma unroll
    for (int e = 0; e < 8; e++) {
        int8_t hi, lo;
        bound_code(mx[e], mn[e], B, hi, lo);
        w[0][e >> 2] |= (uint32_t)(uint8_t)hi << (8 * (e & 3));
        w[1][e >> 2] |= (uint32_t)(uint8_t)lo << (8 * (e & 3));
    }
    uint8_t* b = c.bounds + (size_t)page * c.bblk;
#pragma unroll
    for (int q = 0; q < 2; q++)
        *(uint2*)(b + head * 2 * D + (2 * q + ((g & 3) >> 1)) * (D / 2) + 16 * (g >> 2) + 8 * (g & 1)) =
            make_uint2(w[q][0], w[q][1]);
    if ((g & 3) == 0) *(float*)(b + c.nKV * 2 * D + (head * NG + (g >> 2)) * 4) = B;
}

template <int D>
static hipError_t append_d(hipStream_t st, dim3 grid, bool vec, const CacheDev& c, const OpJobs& jobs, const float* k,
                           int64_t ldk, const float* v, int64_t ldv, int only) {
    return op_launch(vec ? k_kv_append<D, true> : k_kv_append<D, false>, grid, dim3(256), st, c, jobs, k, ldk, v, ldv, only);
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

hipError_t launch_kv_append(hipStream_t st, const CacheDev& c, const OpJobs& jobs, const float* k, int64_t ldk,
                            const float* v, int64_t ldv) {
    const bool vec = aligned16(k) && aligned16(v) && aligned16(c.rope) && ldk % 4 == 0 && ldv % 4 == 0 && c.rot % 16 == 0;
    const dim3 grid(jobs.units, c.nKV, 2);
    if (c.D == 64) return append_d<64>(st, grid, vec, c, jobs, k, ldk, v, ldv, 0);
    if (c.D == 128) return append_d<128>(st, grid, vec, c, jobs, k, ldk, v, ldv, 0);
    return append_d<256>(st, grid, vec, c, jobs, k, ldk, v, ldv, 0);
}

hipError_t launch_kv_bounds(hipStream_t st, const CacheDev& c, const OpJobs& jobs) {
    const dim3 grid(jobs.units, c.nKV, 1);
    if (c.D == 64) return append_d<64>(st, grid, false, c, jobs, nullptr, 0, nullptr, 0, 1);
    if (c.D == 128) return append_d<128>(st, grid, false, c, jobs, nullptr, 0, nullptr, 0, 1);
    return append_d<256>(st, grid, false, c, jobs, nullptr, 0, nullptr, 0, 1);
}

// ========================================================== selected pages ===
// Order-preserving bits of an f32.
__device__ static inline uint32_t order_bits(float v) {
    const uint32_t b = f2u(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// A workgroup's unit of work: part `part` of a row and head. Workgroups go
// round the eight XCDs in launch order, each with its own L2, so an XCD gets
// a run of the units in (head, row, part) order: the rows of a job, which
// read the same bounds and many of the same pages, meet in one L2. row < 0: none.
struct OpWork {
    int row, head, part;
};
__device__ static inline OpWork op_work(int rows, int heads, int parts) {
    const int per = (int)gridDim.x >> 3, w = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
    OpWork o{-1, 0, 0};
    if (w >= rows * heads * parts) return o;
    o.part = w % parts;
    o.row = (w / parts) % rows;
    o.head = w / parts / rows;
    return o;
}
static int op_blocks(int64_t units) { return (int)((units + 7) / 8 * 8); }

// The score of a page for a row and kv head: an upper bound, in 8 bits, of
// q . k over the page's keys, the largest over the head's query heads:
//   sum_b T_b * B_b * (sum_{d in b} qc > 0 ? qc * hi : qc * lo),
// qc, T the query in 8 bits per 32 channels as a key is stored, hi, lo, B the
// page's key bounds. With the query's positive codes beside its negative ones
// the inner sum of a 32-channel group is one 64-wide dot product, [q+ | q-] .
// [hi | lo]: one v_mfma_i32_16x16x64_i8 for 16 query heads and 16 pages, exact.
// The groups' sums meet in f64 (T * B is exact there), and the score is that
// sum rounded to f32, so which pages a row keeps does not depend on an order
// of summation. Kept as the score's order-preserving bits.
//
// A wave takes a tile of 16 pages, the 4 waves of a workgroup 64 pages one
// after another of one row and kv head, reading 2*D + 4*D/32 bytes a page. (Two
// tiles a wave: the same at head_dim 128, 128 verify rows at 256 3% slower.)
// The rows of a job read the same bounds (op_work puts them on one L2). 32 rows
// of 4096 to 32768 tokens, 8 kv heads of 128 (20 MB of bounds): 12.6 us, in
// which a workgroup waits for one load after another (job, page, bounds); held
// to registers for more waves a SIMD its own loads wait too, and 5 waves take
// 5 us more.
constexpr int SCORE_PAGES = 64;
template <int NG>
__global__ __launch_bounds__(256) void k_page_score(CacheDev c, OpJobs jobs, AttendPlan p, const float* __restrict__ q,
                                                    int64_t ldq, uint32_t* __restrict__ scores,
                                                    uint32_t* __restrict__ counters, int n_counters) {
    constexpr int D = 32 * NG;
    __shared__ __align__(16) int8_t qc[16][D];
    __shared__ float qs[16][NG];
    // the attention launch that follows counts its finished workgroups
    for (int i = blockIdx.x * 256 + threadIdx.x; i < n_counters; i += gridDim.x * 256) counters[i] = 0;
    const OpWork wk = op_work(jobs.rows, c.nKV, p.score_blocks);
    const int row = wk.row, kvh = wk.head;
    if (row < 0) return;
    const OpJob jb = job_of(jobs, row);
    const int pos = jb.past + row - jb.first, seen = (pos >> 6) + 1;
    const int page0 = wk.part * SCORE_PAGES, page1 = seen - p.recent;
    if (seen <= p.budget || page0 >= page1 || page0 + SCORE_PAGES <= p.sink) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, kb = lane >> 4;
    const uint32_t* pt = c.page_table + (size_t)jb.slot * c.max_pages;
    const float* cs = c.rope + (size_t)pos * c.rot;
    const float* qr = q + (jb.row0 + row - jb.first) * ldq + (size_t)kvh * p.group * D;
    const int page = page0 + wave * 16 + l16;
    const uint32_t id = page < page1 ? pt[page] : 0u;
    const bool there = id < (uint32_t)c.n_pages;   // a page index outside the cache: never kept for its score
    u32x4 b[NG];
    float B[NG];
    {
        const uint8_t* at = c.bounds + (size_t)(there ? id : 0u) * c.bblk;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            b[g] = *(const u32x4_a4*)(at + kvh * 2 * D + kb * (D / 2) + 16 * g);
            B[g] = *(const float*)(at + c.nKV * 2 * D + (kvh * NG + g) * 4);
        }
    }
    float best = -INFINITY;
    for (int h0 = 0; h0 < p.group; h0 += 16) {
        const int gt = min(16, p.group - h0);
        if (h0) __syncthreads();
        for (int i = threadIdx.x; i < gt * (D / 8); i += 256) {   // 8 channels a thread, a group of 32 in 4 lanes
            const int h = i / (D / 8), d0 = 8 * (i & (D / 8 - 1));
            float r[8];
            rotated8(qr + (size_t)(h0 + h) * D, d0, cs, c.rot, p.vec, r);
            float amax = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(r[e]));
            amax = fmaxf(amax, __shfl_xor(amax, 1));
            amax = fmaxf(amax, __shfl_xor(amax, 2));
            const float scale = amax / 127.0f;
            const float inv = scale > 0.0f ? 1.0f / scale : 0.0f;
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; e++)
                w[e >> 2] |= (uint32_t)(uint8_t)(int8_t)(int)fminf(fmaxf(__builtin_rintf(r[e] * inv), -127.0f), 127.0f)
                             << (8 * (e & 3));
            *(uint2*)&qc[h][d0] = make_uint2(w[0], w[1]);
            if ((d0 & 31) == 0) qs[h][d0 >> 5] = scale;
        }
        __syncthreads();
        // the lane's operand: head l16, codes 32g + 16(kb % 2) .., the positive (kb < 2) or the negative ones;
        // rows of heads past the tile's come from whatever lies there, and are left out below
        double acc[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const u32x4 w = *(const u32x4*)&qc[l16][32 * g + 16 * (kb & 1)];
            u32x4 a;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t neg = ((w[e] >> 7) & 0x01010101u) * 0xffu;
                a[e] = w[e] & (kb < 2 ? ~neg : neg);
            }
            i32x4 d = {0, 0, 0, 0};
            d = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b[g]), d, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; r++) acc[r] = fma((double)qs[4 * kb + r][g] * (double)B[g], (double)d[r], acc[r]);
        }
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (4 * kb + r < gt) best = fmaxf(best, (float)acc[r]);
    }
    best = fmaxf(best, __shfl_xor(best, 16));
    best = fmaxf(best, __shfl_xor(best, 32));
    if (kb == 0 && page < page1)
        scores[((size_t)row * c.nKV + kvh) * p.max_seen + page] = order_bits(there ? best : -INFINITY);
}

// The pages that a row and kv head keep, ascending: entries [e0, e1) of them
// into list (LDS). Entry order: the first `sink` pages, the `need` best of the
// pages [a, z) by score (ties to the lower page), the last `recent`. The
// `need`-th largest score comes from four passes over its bits from the top,
// 8 at a time, with a count of the scores that share the bits so far; then
// every thread ranks a run of pages. KEEP: a thread's run is at most
// SELECT_REG pages, held in registers throughout.
// Up to 256 pages (one a thread) are ranked by counting instead: the larger
// keys out of LDS, no passes (of 141 pages: 2.4 us instead of 3.9).
// mine, id: page a + threadIdx.x's score and index in the cache.
__device__ static inline void best_few_pages(uint32_t mine, uint32_t id, int a, int n, uint32_t need, int sink, int e0, int e1,
                                             uint16_t* list, uint32_t* ids, uint64_t* keys, uint32_t* s_sel) {
    const int t = threadIdx.x, wave = t >> 6;
    const uint64_t key = t < n ? (uint64_t)mine << 32 | (uint32_t)(255 - t) : 0;   // unique: the lower page is the larger
    keys[t] = key;
    __syncthreads();
    uint32_t rank = 0;
    for (int i = 0; i < n; i += 8) {   // past n: zeros, larger than none
        ulonglong2 k[4];
#pragma unroll
        for (int e = 0; e < 4; e++) k[e] = *(const ulonglong2*)(keys + i + 2 * e);
#pragma unroll
        for (int e = 0; e < 4; e++) rank += (k[e].x > key) + (k[e].y > key);
    }
    const bool keep = t < n && rank < need;
    const uint64_t in = __ballot(keep);
    if ((t & 63) == 0) s_sel[wave] = (uint32_t)__popcll(in);
    __syncthreads();
    int e = sink + __popcll(in & ((1ull << (t & 63)) - 1));
    for (int w = 0; w < wave; w++) e += (int)s_sel[w];
    if (keep && e >= e0 && e < e1) {
        list[e - e0] = (uint16_t)(a + t);
        ids[e - e0] = id;
    }
}

constexpr int SELECT_REG = 4;
template <bool KEEP>
__device__ static inline void best_pages(const uint32_t* __restrict__ sc, int a, int z, uint32_t need, int sink, int e0,
                                         int e1, const uint32_t* __restrict__ pt, uint16_t* list, uint32_t* ids,
                                         uint32_t* hist, uint32_t* s_sel) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int per = KEEP ? SELECT_REG : (z - a + 255) / 256, i0 = a + t * per, i1 = min(i0 + per, z);
    uint32_t reg[SELECT_REG];
    if (KEEP)
#pragma unroll
        for (int e = 0; e < SELECT_REG; e++) reg[e] = i0 + e < i1 ? sc[i0 + e] : 0u;
    auto each = [&](auto&& f) {
        if (KEEP) {
#pragma unroll
            for (int e = 0; e < SELECT_REG; e++)
                if (i0 + e < i1) f(i0 + e, reg[e]);
        } else {
            for (int i = i0; i < i1; i++) f(i, sc[i]);
        }
    };
    uint32_t prefix = 0, left = need;
    for (int sh = 24; sh >= 0; sh -= 8) {
        hist[t] = 0;
        __syncthreads();
        each([&](int, uint32_t k) {
            if (sh == 24 || (k >> (sh + 8)) == (prefix >> (sh + 8))) atomicAdd(&hist[(k >> sh) & 255u], 1u);
        });
        __syncthreads();
        if (wave == 0) {
            // lane l: digits 255 - 4l .. 252 - 4l, from the largest down
            uint32_t n[4], sum = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                n[e] = hist[255 - 4 * lane - e];
                sum += n[e];
            }
            uint32_t before = sum;
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t x = __shfl_up(before, o);
                if (lane >= o) before += x;
            }
            before -= sum;
            if (before < left && left <= before + sum) {
                int e = 0;
                while (before + n[e] < left) before += n[e++];
                s_sel[0] = prefix | ((uint32_t)(255 - 4 * lane - e) << sh);
                s_sel[1] = left - before;
            }
        }
        __syncthreads();
        prefix = s_sel[0];
        left = s_sel[1];
    }
    // prefix: the need-th largest score's bits; `left` of the pages that have them are kept
    uint32_t gt = 0, eq = 0;
    each([&](int, uint32_t k) {
        gt += k > prefix;
        eq += k == prefix;
    });
    uint32_t bg = gt, be = eq;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(bg, o), y = __shfl_up(be, o);
        if (lane >= o) {
            bg += x;
            be += y;
        }
    }
    if (lane == 63) {
        hist[wave] = bg;
        hist[4 + wave] = be;
    }
    __syncthreads();
    bg -= gt;
    be -= eq;
    for (int w = 0; w < wave; w++) {
        bg += hist[w];
        be += hist[4 + w];
    }
    each([&](int i, uint32_t k) {
        if (k > prefix || (k == prefix && be < left)) {
            const int e = sink + (int)(bg + min(be, left));
            if (e >= e0 && e < e1) {
                list[e - e0] = (uint16_t)i;
                ids[e - e0] = pt[i];
            }
        }
        bg += k > prefix;
        be += k == prefix;
    });
}

// Attention of a row's query heads (a tile of up to 16 of one kv head's) over
// its kept pages, split over workgroups of `per` pages and those over four
// waves. A wave walks its pages as the pass's attention does (online softmax
// in log2 units; S^T = K . Q^T with the query as an f16 pair; O^T += V^T .
// (p * s) with p * s as an f16 pair; one page of codes in flight), but its
// pages come from a list, and a page's V scales enter p * s relative to the
// power of two below the largest of their 32-channel group, so that f16 holds
// them whatever the values' magnitude, also where it differs from group to
// group (O's channels of a group are carried relative to the last page's). The waves'
// parts meet in LDS, the workgroups' in the workspace: the last workgroup of a
// (row, tile) to finish joins them in split order, whichever it is, so a row's
// result does not depend on it.
//
// 32 rows, 8 kv heads of 128, 64 pages each (302 MB): 61 us, 4.9 TB/s, memory.
// 128 rows, 4 heads of 256, 48 pages: 149 us, one wave a SIMD. A page is some
// 1490 vector instructions (codes unpacked, P split) and 128 MFMA, 24 pages a
// SIMD 60-80 us of them; the rest is waiting that one wave does not cover. It
// holds 256 registers and 144 in the accumulation file; two waves have 256 in
// all each, where it spills and takes twice as long.
// Rows of a prompt take a tile each as well: 512 rows at 8192 of 40 heads of
// 128, 64 pages a row, 0.6 ms.
// One row, 8 heads of 128, 32 pages: 14 us, a chain of choice (2.4 of it),
// pages and two joins.
template <int NG>
__global__ __launch_bounds__(256, NG > 4 ? 1 : 2) void k_attend_pages(CacheDev c, OpJobs jobs, AttendPlan p,
                                                                      const float* __restrict__ q, int64_t ldq,
                                                                      const uint32_t* __restrict__ scores,
                                                                      float* __restrict__ partials,
                                                                      uint32_t* __restrict__ counters,
                                                                      float* __restrict__ out, int64_t ldo) {
    constexpr int D = 32 * NG, DT = D / 16, SCL = NG > 4 ? NG / 4 : 1;
    constexpr int OW = 16 * D + 32;   // floats of a wave's part: O [16][D], max [16], sum [16]
    __shared__ __align__(16) float smem[ATTEND_WAVES * OW];
    __shared__ uint16_t list[ATTEND_PER];   // the kept pages, and their indices in the cache
    __shared__ uint32_t ids[ATTEND_PER];
    __shared__ __align__(16) uint32_t hist[512];
    __shared__ uint32_t s_sel[4];
    static_assert(ATTEND_WAVES * OW >= 2 * 16 * ATTEND_SPLITS, "the join's weights take the parts' place");
    const OpWork wk = op_work(jobs.rows, c.nKV * p.tiles, p.splits);
    const int row = wk.row, split = wk.part, kvh = wk.head / p.tiles, tile = wk.head % p.tiles;
    if (row < 0) return;
    const OpJob jb = job_of(jobs, row);
    const int pos = jb.past + row - jb.first, seen = (pos >> 6) + 1;
    const int kept = min(seen, p.budget);
    const int splits = (kept + p.per - 1) / p.per;   // of this row
    if (split >= splits) return;
    const int e0 = split * p.per, e1 = min(e0 + p.per, kept);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, j4 = lane >> 4, l16 = lane & 15;
    const int h0 = tile * 16, gt = min(16, p.group - h0);
    const uint32_t* pt = c.page_table + (size_t)jb.slot * c.max_pages;
    // what the kept pages are found from, in flight while the query is rotated
    const int a = p.sink, z = seen - p.recent, need = p.budget - p.sink - p.recent;
    const uint32_t* sc = scores + ((size_t)row * c.nKV + kvh) * p.max_seen;
    const bool few = seen > p.budget && need > 0 && z - a <= 256;
    const uint32_t few_score = few && tid < z - a ? sc[a + tid] : 0u, few_id = few && tid < z - a ? pt[a + tid] : 0u;
    // the other entries: the first and the last pages, or all of them
    int end_page = -1;
    uint32_t end_id = 0;
    if (tid < e1 - e0) {
        const int e = e0 + tid;
        if (seen <= p.budget || e < a) end_page = e;
        else if (e >= a + need) end_page = z + e - a - need;
        if (end_page >= 0) end_id = pt[end_page];
    }
    // the query heads, rotated, in LDS (a wave's scale slices and part come there later)
    {
        const float* cs = c.rope + (size_t)pos * c.rot;
        const float* qr = q + (jb.row0 + row - jb.first) * ldq + (size_t)(kvh * p.group + h0) * D;
        for (int i = tid; i < gt * (D / 8); i += 256) {
            const int h = i / (D / 8), d0 = 8 * (i & (D / 8 - 1));
            float r[8];
            rotated8(qr + (size_t)h * D, d0, cs, c.rot, p.vec, r);
            *(float4*)&smem[h * D + d0] = make_float4(r[0], r[1], r[2], r[3]);
            *(float4*)&smem[h * D + d0 + 4] = make_float4(r[4], r[5], r[6], r[7]);
        }
    }
    if (end_page >= 0) {
        list[tid] = (uint16_t)end_page;
        ids[tid] = end_id;
    }
    if (few) best_few_pages(few_score, few_id, a, z - a, need, a, e0, e1, list, ids, (uint64_t*)hist, s_sel);
    else if (seen > p.budget && need > 0) {
        if (z - a <= 256 * SELECT_REG) best_pages<true>(sc, a, z, need, a, e0, e1, pt, list, ids, hist, s_sel);
        else best_pages<false>(sc, a, z, need, a, e0, e1, pt, list, ids, hist, s_sel);
    }
    __syncthreads();
    // this wave's entries of the list, one a lane
    const int n = e1 - e0, w0 = (n * wave) / ATTEND_WAVES, w1 = (n * (wave + 1)) / ATTEND_WAVES, nw = w1 - w0;
    const int lp = lane < nw ? (int)list[w0 + lane] : 0;
    const uint32_t pgv = lane < nw ? ids[w0 + lane] : 0u;
    // the lane's head (none past the tile's: zero) as an f16 pair, with its largest value brought to 2^3 .. 2^4 by a power
    // of two, so that f16 holds it whatever the query's magnitude; the scores take the power back
    float qmax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8 * NG; i += 4) {
        const float4 f = *(const float4*)&smem[l16 * D + 32 * (i >> 3) + 8 * j4 + (i & 4)];
        qmax = fmaxf(qmax, fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w))));
    }
    qmax = fmaxf(qmax, __shfl_xor(qmax, 16));
    qmax = fmaxf(qmax, __shfl_xor(qmax, 32));
    const int eq = max((int)(f2u(qmax) >> 23) - 127, -120) - 3;
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
                split_hilo(l16 < gt ? x[i] * qdown : 0.0f, hi, lo);
                qh[g][e + i] = hi;
                ql[g][e + i] = lo;
            }
        }
    __syncthreads();   // every wave has its query: the space is free
    float* ksl = smem + wave * OW;
    float* vsl = ksl + 256 * SCL;
    const float score_scale = 1.4426950408889634f / sqrtf((float)D) * u2f((uint32_t)(127 + eq) << 23);
    const size_t pstride = (size_t)c.nKV * c.blk, hoff = (size_t)kvh * c.blk;
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
    float mrow = -INFINITY, lsum = 0.0f;
    bool shifted = true;   // p carries 2^PV_SHIFT_LOG2 until a running max leaves no room for it
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
        const int p64 = 64 * __builtin_amdgcn_readlane(lp, i);
        const bool bad = (uint32_t)__builtin_amdgcn_readlane(pgv, i) >= (uint32_t)c.n_pages;
        const int last = bad ? -1 : pos;   // the last token that counts
        // a group's V scales are one row of 16 lanes: the exponent of the largest (all zero: as before), and every scale
        // relative to it; O has room for values 2^60 times as large as this page's
        int by[SCL];   // what brings O from the page before to this one's exponent
#pragma unroll
        for (int s = 0; s < SCL; s++) {
            *(u32x4*)&ksl[256 * s + lane * 4] = kst[s];
            if (p64 + 63 > last) {   // tokens past the row: whatever scale lies there, NaN too, goes in as zero
                const int t0 = p64 + 16 * (lane & 3) + 4 * (((256 * s + lane * 4) >> 4) & 3);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (t0 + e > last) vst[s][e] = 0u;
            }
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) top = max(top, vst[s][e]);   // scales are not negative
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
                const u32x4 w = kc[tt][g >> 1];
                const half8_t kf = (g & 1) ? dequant8_biased(w[2], w[3]) : dequant8_biased(w[0], w[1]);
                float4_t pp = {0.f, 0.f, 0.f, 0.f};
                pp = mfma16x16x32(kf, qh[g], pp);
                pp = mfma16x16x32(kf, ql[g], pp);
#pragma unroll
                for (int r = 0; r < 4; r++) acc[r] = __builtin_fmaf(ks[r * NG + g], pp[r], acc[r]);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) pr[tt][r] = acc[r] * score_scale;
        }
        if (p64 + 63 > last) {
#pragma unroll
            for (int tt = 0; tt < 4; tt++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (p64 + tt * 16 + 4 * j4 + r > last) pr[tt][r] = -INFINITY;
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
        const float mnew = fmaxf(mrow, pm);
        const bool drop = !(fabsf(mnew) < PV_MAX_SCORE) && mnew != -INFINITY;   // -inf: nothing but masked tokens yet
        const float shrink = drop && shifted ? PV_UNSHIFT : 1.0f;
        shifted = shifted && !drop;
        const float alpha = (mrow == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mrow - mnew)) * shrink;
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
        const float msub = (mnew == -INFINITY ? 0.0f : mnew) - (shifted ? PV_SHIFT_LOG2 : 0.0f);
#pragma unroll
        for (int tt = 0; tt < 4; tt++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float e = __builtin_amdgcn_exp2f(pr[tt][r] - msub);
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
                    uint32_t h, l;
                    split_hilo2(pr[tt][r] * sv[4 * tt + r], pr[tt][r + 1] * sv[4 * tt + r + 1], h, l);
                    phw[ii >> 1] = h;
                    plw[ii >> 1] = l;
                }
                const half8_t ph = __builtin_bit_cast(half8_t, phw), pl = __builtin_bit_cast(half8_t, plw);
#pragma unroll
                for (int dd = 0; dd < 2; dd++) {
                    const int dt = 2 * b + dd;
                    const u32x4 w = vc[dt];
                    const half8_t vf = ks ? dequant8_biased(w[2], w[3]) : dequant8_biased(w[0], w[1]);
                    o[dt] = mfma16x16x32(vf, ph, o[dt]);
                    o[dt] = mfma16x16x32(vf, pl, o[dt]);
                }
            }
        }
        mrow = mnew;
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
        const float un = shifted ? PV_UNSHIFT : 1.0f;
        float* part = smem + wave * OW;   // its scale slices are this wave's own and done with
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
            *(float4_t*)(part + l16 * D + dt * 16 + 4 * j4) =
                o[dt] * ldexpf(un, __builtin_amdgcn_readlane(ev[dt >> 3], 16 * ((dt >> 1) & 3)));
        if (j4 == 0) {
            part[16 * D + l16] = mrow;
            part[16 * D + 16 + l16] = lsum * un;
        }
    }
    __syncthreads();
    // the four waves' parts of the tile's heads, two channels a thread
    float* dst = out + (jb.row0 + row - jb.first) * ldo + (size_t)(kvh * p.group + h0) * D;
    const size_t unit = ((size_t)row * c.nKV + kvh) * p.tiles + tile;
    const int gw = min(16, p.group);
    const size_t part_floats = (size_t)gw * (D + 2);   // of a split: O [gw][D], then (max, sum) [gw]
    float* mine = partials + (unit * p.splits + split) * part_floats;
    for (int i = tid; i < gt * (D / 2); i += 256) {
        const int h = i / (D / 2), d = 2 * (i & (D / 2 - 1));
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < ATTEND_WAVES; w++) m = fmaxf(m, smem[w * OW + 16 * D + h]);
        const float ms = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
        for (int w = 0; w < ATTEND_WAVES; w++) {
            const float* part = smem + w * OW;
            const float f = __builtin_amdgcn_exp2f(part[16 * D + h] - ms);
            const float2 xy = *(const float2*)(part + h * D + d);
            l = __builtin_fmaf(part[16 * D + 16 + h], f, l);
            x = __builtin_fmaf(xy.x, f, x);
            y = __builtin_fmaf(xy.y, f, y);
        }
        if (splits == 1) {
            dst[(size_t)h * D + d] = l != 0.0f ? x / l : 0.0f;
            dst[(size_t)h * D + d + 1] = l != 0.0f ? y / l : 0.0f;
        } else {
            leave64(mine + (size_t)h * D + d, (unsigned long long)f2u(y) << 32 | f2u(x));
            if (d == 0) leave64(mine + (size_t)gw * D + 2 * h, (unsigned long long)f2u(l) << 32 | f2u(m));
        }
    }
    if (splits == 1) return;
    if (!finished_last(&counters[unit], splits, s_sel)) return;
    // the splits' weights: 16 threads a head, over its splits
    const float* all = partials + unit * p.splits * part_floats;
    float* wt = smem;                          // [splits][16]
    float* total = smem + 16 * ATTEND_SPLITS;  // [16]
    {
        const int h = tid >> 4, s0 = tid & 15;
        float m[ATTEND_SPLITS / 16], l[ATTEND_SPLITS / 16], mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < ATTEND_SPLITS / 16; e++) {
            const int s = s0 + 16 * e;
            const unsigned long long v =
                h < gt && s < splits ? left64(all + s * part_floats + (size_t)gw * D + 2 * h) : (unsigned long long)f2u(-INFINITY);
            m[e] = u2f((uint32_t)v);
            l[e] = u2f((uint32_t)(v >> 32));
            mx = fmaxf(mx, m[e]);
        }
        for (int x = 1; x < 16; x <<= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
        const float ms = mx == -INFINITY ? 0.0f : mx;
        // the sum in split order within a thread's splits, then across the threads: an order of its own, always the same
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < ATTEND_SPLITS / 16; e++) {
            const float f = __builtin_amdgcn_exp2f(m[e] - ms);
            sum = __builtin_fmaf(l[e], f, sum);
            if (s0 + 16 * e < splits) wt[(s0 + 16 * e) * 16 + h] = f;
        }
        for (int x = 1; x < 16; x <<= 1) sum += __shfl_xor(sum, x);
        if (s0 == 0) total[h] = sum;
    }
    __syncthreads();
    for (int i = tid; i < gt * (D / 2); i += 256) {
        const int h = i / (D / 2), d = 2 * (i & (D / 2 - 1));
        const float* part = all + (size_t)h * D + d;
        float x = 0.0f, y = 0.0f;
        for (int s = 0; s < splits; s += 8) {   // eight loads in flight
            unsigned long long v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = s + e < splits ? left64(part + (size_t)(s + e) * part_floats) : 0ull;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float f = s + e < splits ? wt[(s + e) * 16 + h] : 0.0f;
                x = __builtin_fmaf(u2f((uint32_t)v[e]), f, x);
                y = __builtin_fmaf(u2f((uint32_t)(v[e] >> 32)), f, y);
            }
        }
        const float l = total[h];
        dst[(size_t)h * D + d] = l != 0.0f ? x / l : 0.0f;
        dst[(size_t)h * D + d + 1] = l != 0.0f ? y / l : 0.0f;
    }
}

template <int NG>
static hipError_t attend_ng(hipStream_t st, const CacheDev& c, const OpJobs& jobs, const AttendPlan& p, const float* q,
                            int64_t ldq, float* out, int64_t ldo, uint8_t* ws) {
    uint32_t* scores = (uint32_t*)(ws + p.scores);
    float* partials = (float*)(ws + p.partials);
    uint32_t* counters = (uint32_t*)(ws + p.counters);
    if (p.scored || p.splits > 1) {
        const int n_counters = p.splits > 1 ? jobs.rows * c.nKV * p.tiles : 0;
        const hipError_t e = op_launch(k_page_score<NG>, dim3(op_blocks((int64_t)jobs.rows * c.nKV * p.score_blocks)),
                                       dim3(256), st, c, jobs, p, q, ldq, scores, counters, n_counters);
        if (e != hipSuccess) return e;
    }
    return op_launch(k_attend_pages<NG>, dim3(op_blocks((int64_t)jobs.rows * c.nKV * p.tiles * p.splits)), dim3(256), st, c,
                     jobs, p, q, ldq, scores, partials, counters, out, ldo);
}

hipError_t launch_attend_pages(hipStream_t st, const CacheDev& c, const OpJobs& jobs, const AttendPlan& plan,
                               const float* q, int64_t ldq, float* out, int64_t ldo, uint8_t* ws) {
    AttendPlan p = plan;
    p.score_blocks = p.scored ? (p.max_seen - p.recent + SCORE_PAGES - 1) / SCORE_PAGES : 1;
    p.vec = aligned16(q) && aligned16(c.rope) && ldq % 4 == 0 && c.rot % 16 == 0;
    if (c.ng == 2) return attend_ng<2>(st, c, jobs, p, q, ldq, out, ldo, ws);
    if (c.ng == 4) return attend_ng<4>(st, c, jobs, p, q, ldq, out, ldo, ws);
    return attend_ng<8>(st, c, jobs, p, q, ldq, out, ldo, ws);
}
