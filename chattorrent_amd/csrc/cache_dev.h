// Device code that the operators on a paged cache share (cache_ops.hip,
// kept_ops.hip).
#pragma once
#include "common.h"
#include "ops.h"

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));

// The job that holds unit u (uniform: u comes from the block's index).
__device__ static inline int job_at(const OpJobs& jobs, int u) {
    int lo = 0, hi = jobs.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (jobs.j[mid].first <= u) lo = mid;
        else hi = mid;
    }
    return lo;
}
__device__ static inline OpJob job_of(const OpJobs& jobs, int u) { return jobs.j[job_at(jobs, u)]; }

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

// The same at the positions that the call's row `row` is given: pair j turns
// by the position on its axis, one beyond the table by the table's nearest.
__device__ static inline void rotated8_at(const float* __restrict__ x, int d0, const CacheDev& c, const AxesDev& axes,
                                          int64_t row, bool vec, float (&r)[8]) {
    const int half = c.rot >> 1;
    const int32_t* at = axes.pos + row * axes.n;
    const float2* table[4];
#pragma unroll
    for (int a = 0; a < 4; a++)
        table[a] = (const float2*)(c.rope + (size_t)min(max(at[min(a, axes.n - 1)], 0), c.rope_rows - 1) * c.rot);
    auto turn = [&](int j) {   // pair j's cos and sin
        const uint32_t a = axes.of[j >> 4] >> (2 * (j & 15)) & 3u;
        const float2* lo = a & 1u ? table[1] : table[0];
        const float2* hi = a & 1u ? table[3] : table[2];
        return (a & 2u ? hi : lo)[j];
    };
    if (vec) {
        const float4 a = *(const float4*)(x + d0), b = *(const float4*)(x + d0 + 4);
        r[0] = a.x; r[1] = a.y; r[2] = a.z; r[3] = a.w;
        r[4] = b.x; r[5] = b.y; r[6] = b.z; r[7] = b.w;
        if (d0 < c.rot) {
            const bool low = d0 < half;
            const float* y = x + d0 + (low ? half : -half);
            const float4 ya = *(const float4*)y, yb = *(const float4*)(y + 4);
            const float o[8] = {ya.x, ya.y, ya.z, ya.w, yb.x, yb.y, yb.z, yb.w};
            const int j0 = d0 - (low ? 0 : half);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float2 t = turn(j0 + e);
                r[e] = low ? r[e] * t.x - o[e] * t.y : r[e] * t.x + o[e] * t.y;
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int d = d0 + e;
        r[e] = x[d];
        if (d < c.rot) {
            const float2 t = turn(d < half ? d : d - half);
            const float o = x[d < half ? d + half : d - half];
            r[e] = d < half ? r[e] * t.x - o * t.y : r[e] * t.x + o * t.y;
        }
    }
}

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

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

