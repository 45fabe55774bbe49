// Operators on rows of logits in device memory: penalties, biases and grammar
// masks (cc_logits_adjust), and the draw of a token from the adjusted row
// (cc_sample).
#include "common.h"
#include "ops.h"

// ================================================================= adjust ===
// A row's adjusted logits, by chunks of the vocabulary. With c the sum of the
// row's history counts of a token (an entry counts 1 where no counts are
// given):
//   v = x;  c > 0:  v = v > 0 ? v / rep : v * rep;  v -= pres + min(freq * c, cap)
//   + the bias of the token's last entry;  masked out: -inf
// in f64, rounded to f32 once (an untouched token's bits stay as they are).
// The chunk's counts and its tokens' last bias entries are gathered in LDS, so
// an id that occurs twice needs no order: counts add up as integers, and the
// largest entry index wins.
constexpr int LG_T = 256;

struct RowPens {
    double rep, freq, pres, cap;
    int p0, p1, b0, b1;   // the row's entries of the history and the bias list
    const uint32_t* mask; // its words, or null
};
__device__ static inline RowPens row_pens(const SamplingDev& s, int row) {
    RowPens r;
    r.rep = s.rep ? (double)s.rep[row] : 1.0;
    r.freq = s.freq ? (double)s.freq[row] : 0.0;
    r.pres = s.pres ? (double)s.pres[row] : 0.0;
    r.cap = (double)s.freq_cap;
    r.p0 = r.p1 = r.b0 = r.b1 = 0;
    if (s.pen_at) {
        r.p0 = max(s.pen_at[row], 0);
        r.p1 = min(s.pen_at[row + 1], s.n_pen);
    }
    if (s.bias_at) {
        r.b0 = max(s.bias_at[row], 0);
        r.b1 = min(s.bias_at[row + 1], s.n_bias);
    }
    r.mask = nullptr;
    if (s.mask) {
        const int m = s.mask_of[row];
        if (m >= 0 && m < s.n_masks) r.mask = s.mask + (size_t)m * s.mask_words;
    }
    return r;
}

// The chunk [base, base + CH) of the row's lists into LDS: cnt (history
// counts) and last (bias entry + 1), zero where there is none. False (for the
// whole workgroup) if the row has no list. Ends with a barrier.
template <int CH>
__device__ static inline bool gather_lists(const SamplingDev& s, const RowPens& r, int base, int32_t* cnt,
                                           int32_t* last) {
    if (r.p0 >= r.p1 && r.b0 >= r.b1) return false;
    __syncthreads();   // the previous chunk's readers are done
    for (int i = threadIdx.x; i < CH; i += LG_T) cnt[i] = last[i] = 0;
    __syncthreads();
    for (int i = r.p0 + (int)threadIdx.x; i < r.p1; i += LG_T) {
        const uint32_t at = (uint32_t)s.pen_ids[i] - (uint32_t)base;
        const int n = s.pen_counts ? s.pen_counts[i] : 1;
        if (at < (uint32_t)CH && n > 0) atomicAdd(&cnt[at], n);
    }
    for (int i = r.b0 + (int)threadIdx.x; i < r.b1; i += LG_T) {
        const uint32_t at = (uint32_t)s.bias_ids[i] - (uint32_t)base;
        if (at < (uint32_t)CH) atomicMax(&last[at], i - r.b0 + 1);
    }
    __syncthreads();
    return true;
}

__device__ static inline float adjust_one(float x, const SamplingDev& s, const RowPens& r, int cnt, int last) {
    if (cnt <= 0 && last <= 0) return x;
    double v = (double)x;
    if (cnt > 0) {
        v = v > 0.0 ? v / r.rep : v * r.rep;
        v -= r.pres + fmin(r.freq * (double)cnt, r.cap);
    }
    if (last > 0) v += (double)s.bias[r.b0 + last - 1];
    return (float)v;
}

// A chunk is LG_CH tokens, LG_PER a thread: LG_J runs of four, run j of thread
// t at 4 * (LG_T * j + t). a: the chunk's adjusted logits of row x, in that
// order; -inf past the vocabulary and where the mask bars the token. VEC: the
// row's fours of logits are 16-byte aligned.
constexpr int LG_CH = 4096, LG_J = LG_CH / (4 * LG_T);
template <bool VEC>
__device__ static inline void adjusted_chunk(const float* __restrict__ x, int V, const SamplingDev& s, const RowPens& r,
                                             int base, int32_t* cnt, int32_t* last, float (&a)[LG_J][4]) {
#pragma unroll
    for (int j = 0; j < LG_J; j++) {
        const int t = base + 4 * (LG_T * j + (int)threadIdx.x);
        if (VEC && t + 3 < V) {
            const float4 f = *(const float4*)(x + t);
            a[j][0] = f.x; a[j][1] = f.y; a[j][2] = f.z; a[j][3] = f.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) a[j][e] = t + e < V ? x[t + e] : -INFINITY;
        }
    }
    uint32_t bits[LG_J];
#pragma unroll
    for (int j = 0; j < LG_J; j++) {
        const int t = base + 4 * (LG_T * j + (int)threadIdx.x);
        bits[j] = !r.mask ? 15u : t < V ? r.mask[t >> 5] >> (t & 31) : 0u;
    }
    if (gather_lists<LG_CH>(s, r, base, cnt, last)) {
#pragma unroll
        for (int j = 0; j < LG_J; j++) {
            const int i = 4 * (LG_T * j + (int)threadIdx.x);
            const int4 c = *(const int4*)(cnt + i), l = *(const int4*)(last + i);
            a[j][0] = adjust_one(a[j][0], s, r, c.x, l.x);
            a[j][1] = adjust_one(a[j][1], s, r, c.y, l.y);
            a[j][2] = adjust_one(a[j][2], s, r, c.z, l.z);
            a[j][3] = adjust_one(a[j][3], s, r, c.w, l.w);
        }
    }
#pragma unroll
    for (int j = 0; j < LG_J; j++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (!((bits[j] >> e) & 1u)) a[j][e] = -INFINITY;
}

template <bool VEC>
__global__ __launch_bounds__(LG_T) void k_logits_adjust(const float* x, int64_t ldx, int V, SamplingDev s, float* out,
                                                        int64_t ldo) {
    __shared__ __align__(16) int32_t cnt[LG_CH], last[LG_CH];
    const int row = blockIdx.y, base = blockIdx.x * LG_CH;
    float a[LG_J][4];
    adjusted_chunk<VEC>(x + row * ldx, V, s, row_pens(s, row), base, cnt, last, a);
#pragma unroll
    for (int j = 0; j < LG_J; j++) {
        const int t = base + 4 * (LG_T * j + (int)threadIdx.x);
        float* o = out + row * ldo + t;
        if (VEC && t + 3 < V) {
            *(float4*)o = make_float4(a[j][0], a[j][1], a[j][2], a[j][3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (t + e < V) o[e] = a[j][e];
        }
    }
}

static bool vec_rows(const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 4 == 0; }

hipError_t launch_logits_adjust(hipStream_t st, const float* x, int64_t ldx, int rows, int V, const SamplingDev& s,
                                float* out, int64_t ldo) {
    const dim3 grid((V + LG_CH - 1) / LG_CH, rows);
    if (vec_rows(x, ldx) && vec_rows(out, ldo))
        hipLaunchKernelGGL(k_logits_adjust<true>, grid, dim3(LG_T), 0, st, x, ldx, V, s, out, ldo);
    else
        hipLaunchKernelGGL(k_logits_adjust<false>, grid, dim3(LG_T), 0, st, x, ldx, V, s, out, ldo);
    return hipGetLastError();
}

// ================================================================= sample ===
// With a the adjusted row (a NaN counts as -inf) and temp > 0:
//   s = f32(a / temp) (a finite value stays finite), m = max s,
//   w = exp(s - m) as a whole number of 2^-42 (f64 exp, rounded once), so that
//   sums of weights are exact integers and do not depend on their order;
//   kept by top-k: s >= the k-th largest s (ties stay);
//   kept by top-p: s >= the largest value t for which the kept weights of
//   s >= t reach p of all kept weights (ties stay);
//   kept by min-p: exp(s - m) >= min_p;
//   token: the first whose running sum of kept weights, in the order of the
//   ids, is above u * sum; prob = exp(s - m) / sum.
// temp <= 0 (or null): the first maximum of a, prob 1. No token left: -1, 0.
//
// A row is cut over workgroups (`span` chunks each), in two or three launches:
//   k_sample_max   every workgroup's largest and smallest value;
//   k_sample_mass  with the row's m known, every workgroup's weight. The last
//                  workgroup of a row to finish knows them all: it finds the
//                  one that the token falls into and the token in it. A row
//                  with top-k or top-p instead gets a histogram of m - s in
//                  SM_BINS bins from every workgroup (counts, weights), and the
//                  last one finds the bins that the cuts fall into;
//   k_sample_cut   (only where a row may have top-k or top-p) the values of
//                  those bins, a few hundred of a row as a rule, are gathered;
//                  the last workgroup takes them 8 bits at a time to the cuts'
//                  exact values, and draws.
// A row whose cut falls among more than SM_CAND values (nearly equal logits) is
// drawn by its last workgroup alone, in passes over the row.
constexpr int SM_BINS = 512, SM_CAND = 8192, SM_CHUNKS = (1 << 20) / LG_CH;
constexpr float SM_REACH = 32.0f;            // the histogram's last bin takes everything below m - 32
constexpr double SM_ONE = 4398046511104.0;   // 2^42: a row of 2^20 tokens sums to at most 2^62
typedef unsigned long long u64;

__device__ static inline float scaled_logit(float a, double inv_temp) {
    if (!(a > -INFINITY)) return -INFINITY;   // NaN too
    if (a == INFINITY) return a;
    const float s = (float)((double)a * inv_temp);
    return fminf(fmaxf(s, -3.4028234663852886e38f), 3.4028234663852886e38f) + 0.0f;   // -0 is 0
}
__device__ static inline double weight(float s, float m) {
    return s == m ? 1.0 : exp((double)s - (double)m);
}
__device__ static inline u64 whole_weight(double w) { return (u64)(w * SM_ONE + 0.5); }

__device__ static inline uint32_t ordered(float v) {
    const uint32_t b = f2u(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ static inline float unordered(uint32_t k) { return u2f((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

__device__ static inline u64 wave_sum64(u64 v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// Over the workgroup, to every thread: the sum, the sum of the threads before, the largest.
__device__ static inline u64 block_sum64(u64 v, u64* red) {
    v = wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}
__device__ static inline u64 block_before64(u64 v, u64* red) {
    u64 inc = v;
    for (int o = 1; o < 64; o <<= 1) {
        const u64 y = __shfl_up(inc, o);
        if ((int)(threadIdx.x & 63) >= o) inc += y;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = inc;
    __syncthreads();
    for (int w = 0; w < (int)(threadIdx.x >> 6); w++) inc += red[w];
    return inc - v;
}
__device__ static inline u64 block_max64(u64 v, u64* red) {
    for (int o = 32; o > 0; o >>= 1) {
        const u64 y = __shfl_xor(v, o);
        v = y > v ? y : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    const u64 a = red[0] > red[1] ? red[0] : red[1], b = red[2] > red[3] ? red[2] : red[3];
    return a > b ? a : b;
}

// The workspace of a call: per row and workgroup (groups of them) the largest
// key and the smallest value, the weight, the histogram; per row what the cuts
// found, two counters of finished workgroups and the gathered values.
struct SampleInfo {
    int32_t lo, hi;        // the bins that the cuts fall into
    uint32_t above;        // values in the bins before lo
    uint32_t n_cand;       // gathered values (more than SM_CAND: not all of them were)
    u64 mass_above;        // their weight
    u64 want;              // top-p without top-k: the weight to reach
    uint32_t done[2], pad[2];
};
struct SampleWs {
    u64* best;        // [rows][groups] ordered(a) << 32 | ~token; 0: nothing above -inf
    float* least;     // [rows][groups] the smallest value above -inf
    u64* mass;        // [rows][groups]
    u64* hmass;       // [rows][groups][SM_BINS]
    uint32_t* hcount; // [rows][groups][SM_BINS]
    SampleInfo* info; // [rows]
    uint2* cand;      // [rows][SM_CAND] ordered(s), token
    int groups, span;
};

struct RowAsk {
    double inv, top_p, min_p;
    bool greedy, cut;
    int k;
    __device__ RowAsk(const SamplingDev& s, int row, int V) {
        const double temp = s.temp ? (double)s.temp[row] : 0.0;
        greedy = !(temp > 0.0);
        inv = greedy ? 1.0 : 1.0 / temp;
        k = s.top_k ? s.top_k[row] : 0;
        if (k >= V || k < 0) k = 0;
        top_p = s.top_p ? (double)s.top_p[row] : 1.0;
        if (!(top_p < 1.0)) top_p = 1.0;
        min_p = s.min_p ? fmin((double)s.min_p[row], 1.0) : 0.0;   // the maximum itself stays
        cut = !greedy && (k > 0 || top_p < 1.0);
    }
};

template <bool VEC>
__global__ __launch_bounds__(LG_T) void k_sample_max(const float* __restrict__ x, int64_t ldx, int V, SamplingDev s,
                                                     SampleWs w) {
    __shared__ __align__(16) int32_t cnt[LG_CH], last[LG_CH];
    __shared__ u64 red[4];
    const int row = blockIdx.y, g = blockIdx.x;
    if (g == 0 && threadIdx.x < sizeof(SampleInfo) / 4) ((uint32_t*)(w.info + row))[threadIdx.x] = 0;
    const RowPens r = row_pens(s, row);
    u64 best = 0;
    uint32_t least = 0xffffffffu;
    for (int c = g * w.span; c < (g + 1) * w.span && c * LG_CH < V; c++) {
        float a[LG_J][4];
        adjusted_chunk<VEC>(x + row * ldx, V, s, r, c * LG_CH, cnt, last, a);
#pragma unroll
        for (int j = 0; j < LG_J; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (!(a[j][e] > -INFINITY)) continue;
                const uint32_t t = c * LG_CH + 4 * (LG_T * j + threadIdx.x) + e, o = ordered(a[j][e] + 0.0f);   // -0 is 0
                const u64 k = ((u64)o << 32) | (0xffffffffu - t);
                best = k > best ? k : best;
                least = o < least ? o : least;
            }
    }
    best = block_max64(best, red);
    const u64 low = block_max64(~(u64)least, red);
    if (threadIdx.x == 0) {
        w.best[(size_t)row * w.groups + g] = best;
        w.least[(size_t)row * w.groups + g] = best ? unordered((uint32_t)~low) : INFINITY;
    }
}

// What a row's workgroups share about its draw.
struct RowDraw {
    float m, bins;      // the largest s; bins per unit of m - s
    u64 key;            // the row's best (k_sample_max)
};
__device__ static inline RowDraw row_draw(const SampleWs& w, int row, const RowAsk& ask, u64* red) {
    u64 best = 0, low = 0;
    for (int i = threadIdx.x; i < w.groups; i += LG_T) {
        const u64 b = w.best[(size_t)row * w.groups + i];
        best = b > best ? b : best;
        const u64 l = ~(u64)ordered(w.least[(size_t)row * w.groups + i]);
        low = l > low ? l : low;
    }
    RowDraw d;
    d.key = block_max64(best, red);
    d.m = scaled_logit(unordered((uint32_t)(d.key >> 32)), ask.inv);
    const float least = scaled_logit(unordered((uint32_t)~block_max64(low, red)), ask.inv);
    const float range = d.m - least;   // inf or NaN with infinities
    d.bins = SM_BINS / (range < SM_REACH ? fmaxf(range, 1e-30f) : SM_REACH);
    return d;
}
__device__ static inline int bin_of(float s, const RowDraw& d) {
    return s == d.m ? 0 : (int)fminf((d.m - s) * d.bins, (float)(SM_BINS - 1));
}

// Draws from the chunk at `base` the token with `left` of the kept weights of
// the chunk before it. Called by the whole workgroup.
template <bool VEC, class K>
__device__ static inline void draw_in_chunk(const float* __restrict__ x, int V, const SamplingDev& s, const RowPens& r,
                                            int base, int32_t* cnt, int32_t* last, u64* red, u64 left, u64 total,
                                            K&& kept, int32_t* id, float* prob) {
    float a[LG_J][4];
    adjusted_chunk<VEC>(x, V, s, r, base, cnt, last, a);
#pragma unroll
    for (int j = 0; j < LG_J; j++) {   // runs of 4 * LG_T tokens, one after another
        u64 mw[4], sum = 0;
        double w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            w[e] = 0.0;
            mw[e] = kept(a[j][e], w[e]) ? whole_weight(w[e]) : 0;
            sum += mw[e];
        }
        u64 before = block_before64(sum, red);
        const u64 run = red[0] + red[1] + red[2] + red[3];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (before <= left && left < before + mw[e]) {
                *id = base + 4 * (LG_T * j + (int)threadIdx.x) + e;
                if (prob) *prob = (float)(w[e] * SM_ONE / (double)total);
            }
            before += mw[e];
        }
        if (left < run) return;   // the same for every thread
        left -= run;
    }
}

__device__ static inline u64 target_of(double u, u64 total) {
    const u64 t = (u64)fmax(u * (double)total, 0.0);
    return t < total - 1 ? t : total - 1;
}

// The last workgroup of a row, with the workgroups' kept weights known: mass
// (this thread's workgroup of the row) -> the token.
template <bool VEC, class K>
__device__ static inline void draw_row(const float* __restrict__ x, int V, const SamplingDev& s, const RowPens& r,
                                       const SampleWs& w, int row, u64 mass, int32_t* cnt, int32_t* last, u64* red,
                                       u64* found, K&& kept, int32_t* id, float* prob) {
    const u64 before = block_before64(mass, red);
    const u64 total = red[0] + red[1] + red[2] + red[3];
    const u64 target = target_of(s.u ? s.u[row] : 0.0, total);
    if (before <= target && target < before + mass) {
        found[0] = threadIdx.x;
        found[1] = target - before;
    }
    __syncthreads();
    int c = (int)found[0] * w.span;
    u64 left = found[1];
    for (int i = 1; i < w.span; i++, c++) {   // the workgroup's chunk that holds it
        float a[LG_J][4];
        adjusted_chunk<VEC>(x, V, s, r, c * LG_CH, cnt, last, a);
        u64 sum = 0;
#pragma unroll
        for (int j = 0; j < LG_J; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                double q;
                if (kept(a[j][e], q)) sum += whole_weight(q);
            }
        sum = block_sum64(sum, red);
        if (left < sum) break;
        left -= sum;
    }
    draw_in_chunk<VEC>(x, V, s, r, c * LG_CH, cnt, last, red, left, total, kept, id, prob);
}

template <bool VEC>
__global__ __launch_bounds__(LG_T) void k_sample_mass(const float* __restrict__ x, int64_t ldx, int V, SamplingDev s,
                                                      SampleWs w, int32_t* __restrict__ ids,
                                                      float* __restrict__ probs) {
    __shared__ __align__(16) int32_t cnt[LG_CH], last[LG_CH];
    __shared__ u64 hmass[SM_BINS], red[4], found[2];
    __shared__ uint32_t hcount[SM_BINS], s_last;
    const int row = blockIdx.y, g = blockIdx.x, tid = threadIdx.x;
    const RowAsk ask(s, row, V);
    const RowDraw d = row_draw(w, row, ask, red);
    float* prob = probs ? probs + row : nullptr;
    if (d.key == 0 || ask.greedy) {
        if (g == 0 && tid == 0) {
            ids[row] = d.key ? (int32_t)(0xffffffffu - (uint32_t)d.key) : -1;
            if (prob) *prob = d.key ? 1.0f : 0.0f;
        }
        return;
    }
    const RowPens r = row_pens(s, row);
    const float* xr = x + row * ldx;
    SampleInfo* info = w.info + row;
    const size_t at = (size_t)row * w.groups + g;
    auto kept = [&](float a, double& q) {
        const float v = scaled_logit(a, ask.inv);
        if (!(v > -INFINITY)) return false;
        q = weight(v, d.m);
        return q >= ask.min_p;
    };
    if (!ask.cut) {
        u64 sum = 0;
        for (int c = g * w.span; c < (g + 1) * w.span && c * LG_CH < V; c++) {
            float a[LG_J][4];
            adjusted_chunk<VEC>(xr, V, s, r, c * LG_CH, cnt, last, a);
#pragma unroll
            for (int j = 0; j < LG_J; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    double q;
                    if (kept(a[j][e], q)) sum += whole_weight(q);
                }
        }
        sum = block_sum64(sum, red);
        if (tid == 0) leave64(&w.mass[at], sum);
        if (!finished_last(&info->done[0], w.groups, &s_last)) return;
        draw_row<VEC>(xr, V, s, r, w, row, tid < w.groups ? left64(&w.mass[(size_t)row * w.groups + tid]) : 0, cnt, last, red,
                      found, kept, ids + row, prob);
        return;
    }
    // the histogram; weights only where top-p needs them
    const bool weigh = ask.top_p < 1.0;
    for (int b = tid; b < SM_BINS; b += LG_T) {
        hmass[b] = 0;
        hcount[b] = 0;
    }
    __syncthreads();
    for (int c = g * w.span; c < (g + 1) * w.span && c * LG_CH < V; c++) {
        float a[LG_J][4];
        adjusted_chunk<VEC>(xr, V, s, r, c * LG_CH, cnt, last, a);
#pragma unroll
        for (int j = 0; j < LG_J; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float v = scaled_logit(a[j][e], ask.inv);
                if (!(v > -INFINITY)) continue;
                const int b = bin_of(v, d);
                atomicAdd(&hcount[b], 1u);
                if (weigh) atomicAdd(&hmass[b], whole_weight(weight(v, d.m)));
            }
    }
    __syncthreads();
    // thread t: bins 2t and 2t + 1
    leave64(&w.hcount[at * SM_BINS + 2 * tid], (u64)hcount[2 * tid + 1] << 32 | hcount[2 * tid]);
    if (weigh) {
        leave64(&w.hmass[at * SM_BINS + 2 * tid], hmass[2 * tid]);
        leave64(&w.hmass[at * SM_BINS + 2 * tid + 1], hmass[2 * tid + 1]);
    }
    if (!finished_last(&info->done[0], w.groups, &s_last)) return;
    u64 n[2] = {0, 0}, ms[2] = {0, 0};
    for (int i0 = 0; i0 < w.groups; i0 += 8) {   // eight workgroups' loads in flight
        u64 c2[8], m2[8][2];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const size_t o = ((size_t)row * w.groups + min(i0 + i, w.groups - 1)) * SM_BINS + 2 * tid;
            c2[i] = left64(&w.hcount[o]);
            m2[i][0] = weigh ? left64(&w.hmass[o]) : 0;
            m2[i][1] = weigh ? left64(&w.hmass[o + 1]) : 0;
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i0 + i < w.groups) {
                n[0] += c2[i] & 0xffffffffu;
                n[1] += c2[i] >> 32;
                ms[0] += m2[i][0];
                ms[1] += m2[i][1];
            }
    }
    const u64 nb = block_before64(n[0] + n[1], red);
    const u64 mb = block_before64(ms[0] + ms[1], red);
    const u64 total = red[0] + red[1] + red[2] + red[3];
    // the bin in which a running sum (of counts or weights) first reaches `want`
    auto reach = [&](u64 before, const u64* v, u64 want) {
        if (tid == 0) found[0] = SM_BINS - 1;
        __syncthreads();
        if (before < want && want <= before + v[0] + v[1]) found[0] = 2 * tid + (before + v[0] < want ? 1 : 0);
        __syncthreads();
        const int b = (int)found[0];
        __syncthreads();
        return b;
    };
    // a sum over the bins before b
    auto ahead = [&](u64 before, const u64* v, int b) {
        if (tid == b >> 1) found[0] = before + ((b & 1) ? v[0] : 0);
        __syncthreads();
        const u64 r2 = found[0];
        __syncthreads();
        return r2;
    };
    int lo = SM_BINS - 1, hi = SM_BINS - 1;
    u64 want = 0, base = total;
    if (ask.k > 0) {
        lo = hi = reach(nb, n, (u64)ask.k);
        base = weigh ? ahead(mb, ms, hi) : 0;   // at least this weight is kept
    }
    if (weigh) {
        want = (u64)fmax(ceil(ask.top_p * (double)base), 1.0);
        const int p = reach(mb, ms, want);
        lo = p < lo ? p : lo;
        if (ask.k == 0) hi = lo;
    }
    const u64 above = ahead(nb, n, lo), mass_above = weigh ? ahead(mb, ms, lo) : 0;
    if (tid == 0) {
        info->lo = lo;
        info->hi = hi;
        info->above = (uint32_t)above;
        info->mass_above = mass_above;
        info->want = want;
    }
}

// The value (as ordered bits, at least `floor`) at which the sum over the
// values from the top first reaches `want`, 8 bits at a time: of(i, key) calls
// are made by `each` for every value with its key and what it adds.
template <class E>
__device__ static inline uint32_t find_cut(u64 want, uint32_t floor, u64* hist, u64* sel, E&& each) {
    uint32_t prefix = 0;
    u64 left = want;
    const int tid = threadIdx.x, lane = tid & 63;
    for (int sh = 24; sh >= 0; sh -= 8) {
        __syncthreads();
        hist[tid] = 0;
        if (tid == 0) {
            sel[0] = prefix;
            sel[1] = left;
        }
        __syncthreads();
        each([&](uint32_t key, u64 adds) {
            if (key >= floor && (sh == 24 || (key >> (sh + 8)) == (prefix >> (sh + 8)))) atomicAdd(&hist[(key >> sh) & 255u], adds);
        });
        __syncthreads();
        if (tid < 64) {   // lane l: digits 255 - 4l .. 252 - 4l
            u64 v[4], sum = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[e] = hist[255 - 4 * lane - e];
                sum += v[e];
            }
            u64 before = sum;
            for (int o = 1; o < 64; o <<= 1) {
                const u64 y = __shfl_up(before, o);
                if (lane >= o) before += y;
            }
            before -= sum;
            if (before < left && left <= before + sum) {
                int e = 0;
                while (before + v[e] < left) before += v[e++];
                sel[0] = prefix | ((uint32_t)(255 - 4 * lane - e) << sh);
                sel[1] = left - before;
            }
        }
        __syncthreads();
        prefix = (uint32_t)sel[0];
        left = sel[1];
    }
    return prefix;   // fewer than `want` in all: 0, everything is kept
}

template <bool VEC>
__global__ __launch_bounds__(LG_T) void k_sample_cut(const float* __restrict__ x, int64_t ldx, int V, SamplingDev s,
                                                     SampleWs w, int32_t* __restrict__ ids, float* __restrict__ probs) {
    __shared__ __align__(16) int32_t lists[2 * LG_CH];   // the history counts and last biases; later the gathered keys
    __shared__ u64 gmass[LG_T], hist[256], red[4], found[2];
    __shared__ uint32_t s_last, s_n, s_at;
    static_assert(SM_CAND <= 2 * LG_CH, "the gathered keys take the lists' place");
    static_assert(SM_CHUNKS <= LG_T, "a thread a workgroup of the row");
    int32_t *cnt = lists, *last = lists + LG_CH;
    const int row = blockIdx.y, g = blockIdx.x, tid = threadIdx.x;
    const RowAsk ask(s, row, V);
    if (!ask.cut) return;
    const RowDraw d = row_draw(w, row, ask, red);
    if (d.key == 0) return;
    const RowPens r = row_pens(s, row);
    const float* xr = x + row * ldx;
    SampleInfo* info = w.info + row;
    const int lo = info->lo, hi = info->hi;
    uint2* cand = w.cand + (size_t)row * SM_CAND;
    u64 sum = 0;
    for (int c = g * w.span; c < (g + 1) * w.span && c * LG_CH < V; c++) {
        float a[LG_J][4];
        adjusted_chunk<VEC>(xr, V, s, r, c * LG_CH, cnt, last, a);
        uint32_t in = 0;
#pragma unroll
        for (int j = 0; j < LG_J; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float v = scaled_logit(a[j][e], ask.inv);
                a[j][e] = v;
                if (!(v > -INFINITY)) continue;
                const int b = bin_of(v, d);
                if (b < lo) {
                    const double q = weight(v, d.m);
                    if (q >= ask.min_p) sum += whole_weight(q);
                } else if (b <= hi) {
                    in |= 1u << (4 * j + e);
                }
            }
        // the workgroup's place among the gathered values, then each thread's
        if (tid == 0) s_n = 0;
        __syncthreads();
        uint32_t mine = in ? atomicAdd(&s_n, (uint32_t)__popc(in)) : 0;
        __syncthreads();
        if (tid == 0 && s_n) s_at = atomicAdd(&info->n_cand, s_n);
        __syncthreads();
        mine += s_at;
#pragma unroll
        for (int j = 0; j < LG_J; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if ((in >> (4 * j + e)) & 1u) {
                    if (mine < SM_CAND)
                        leave64(&cand[mine], (u64)(c * LG_CH + 4 * (LG_T * j + tid) + e) << 32 | ordered(a[j][e]));
                    mine++;
                }
        __syncthreads();
    }
    sum = block_sum64(sum, red);
    if (tid == 0) leave64(&w.mass[(size_t)row * w.groups + g], sum);
    if (!finished_last(&info->done[1], w.groups, &s_last)) return;
    const uint32_t n = left32(&info->n_cand);
    const u64 above = info->above, mass_above = info->mass_above;
    uint32_t cut = 0;
    gmass[tid] = tid < w.groups ? left64(&w.mass[(size_t)row * w.groups + tid]) : 0;
    auto weigh_key = [&](uint32_t key) { return whole_weight(weight(unordered(key), d.m)); };
    if (n <= SM_CAND) {
        uint32_t* keys = (uint32_t*)lists;
        for (uint32_t i = tid; i < n; i += LG_T) keys[i] = left32(&cand[i].x);
        __syncthreads();
        if (ask.k > 0)
            cut = find_cut((u64)ask.k - above, 0, hist, found, [&](auto&& f) {
                for (uint32_t i = tid; i < n; i += LG_T) f(keys[i], 1ull);
            });
        if (ask.top_p < 1.0) {
            u64 want = info->want;
            if (ask.k > 0) {
                u64 in = 0;
                for (uint32_t i = tid; i < n; i += LG_T)
                    if (keys[i] >= cut) in += weigh_key(keys[i]);
                want = (u64)fmax(ceil(ask.top_p * (double)(mass_above + block_sum64(in, red))), 1.0);
            }
            const uint32_t c2 = find_cut(want - mass_above, cut, hist, found, [&](auto&& f) {
                for (uint32_t i = tid; i < n; i += LG_T) f(keys[i], weigh_key(keys[i]));
            });
            cut = c2 > cut ? c2 : cut;
        }
        __syncthreads();
        for (uint32_t i = tid; i < n; i += LG_T) {
            const double q = weight(unordered(keys[i]), d.m);
            if (keys[i] >= cut && q >= ask.min_p)
                atomicAdd(&gmass[left32(&cand[i].y) / (uint32_t)(LG_CH * w.span)], whole_weight(q));
        }
    } else {
        // too many values share the cut's bins: the same, in passes over the row
        const int chunks = (V + LG_CH - 1) / LG_CH;
        auto all = [&](auto&& f) {
            for (int c = 0; c < chunks; c++) {
                float a[LG_J][4];
                adjusted_chunk<VEC>(xr, V, s, r, c * LG_CH, cnt, last, a);
#pragma unroll
                for (int j = 0; j < LG_J; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float v = scaled_logit(a[j][e], ask.inv);
                        if (v > -INFINITY) f(ordered(v), c);
                    }
            }
        };
        if (ask.k > 0)
            cut = find_cut((u64)ask.k, 0, hist, found, [&](auto&& f) { all([&](uint32_t key, int) { f(key, 1ull); }); });
        if (ask.top_p < 1.0) {
            u64 in = 0;
            all([&](uint32_t key, int) {
                if (key >= cut) in += weigh_key(key);
            });
            const u64 want = (u64)fmax(ceil(ask.top_p * (double)block_sum64(in, red)), 1.0);
            const uint32_t c2 = find_cut(want, cut, hist, found, [&](auto&& f) {
                all([&](uint32_t key, int) {
                    if (key >= cut) f(key, weigh_key(key));
                });
            });
            cut = c2 > cut ? c2 : cut;
        }
        __syncthreads();
        gmass[tid] = 0;
        __syncthreads();
        all([&](uint32_t key, int c) {
            const double q = weight(unordered(key), d.m);
            if (key >= cut && q >= ask.min_p) atomicAdd(&gmass[c / w.span], whole_weight(q));
        });
    }
    __syncthreads();
    auto kept = [&](float a, double& q) {
        const float v = scaled_logit(a, ask.inv);
        if (!(v > -INFINITY) || ordered(v) < cut) return false;
        q = weight(v, d.m);
        return q >= ask.min_p;
    };
    draw_row<VEC>(xr, V, s, r, w, row, gmass[tid], cnt, last, red, found, kept, ids + row, probs ? probs + row : nullptr);
}

// Chunks a workgroup takes: one while the call has few workgroups, more where
// that leaves enough of them (fewer workgroups a row to join).
static int sample_span(int rows, int V) {
    const int chunks = (V + LG_CH - 1) / LG_CH;
    int span = 1;
    while (span < 4 && (int64_t)rows * (chunks / (span * 2)) >= 512) span *= 2;
    return span;
}

static size_t sample_layout(int rows, int V, uint8_t* at, SampleWs& w) {
    w.span = sample_span(rows, V);
    const int chunks = (V + LG_CH - 1) / LG_CH;
    w.groups = (chunks + w.span - 1) / w.span;
    size_t n = 0;
    auto take = [&](size_t bytes) {
        uint8_t* p = at ? at + n : nullptr;
        n += (bytes + 255) & ~(size_t)255;
        return p;
    };
    const size_t gr = (size_t)rows * w.groups;
    w.best = (u64*)take(gr * 8);
    w.least = (float*)take(gr * 4);
    w.mass = (u64*)take(gr * 8);
    w.hmass = (u64*)take(gr * SM_BINS * 8);
    w.hcount = (uint32_t*)take(gr * SM_BINS * 4);
    w.info = (SampleInfo*)take((size_t)rows * sizeof(SampleInfo));
    w.cand = (uint2*)take((size_t)rows * SM_CAND * 8);
    return n;
}

size_t sample_workspace(int rows, int V) {
    SampleWs w;
    return sample_layout(rows, V, nullptr, w);
}

template <bool VEC>
static void sample_vec(hipStream_t st, const float* x, int64_t ldx, int rows, int V, const SamplingDev& s, int32_t* ids,
                       float* probs, const SampleWs& w) {
    const dim3 grid(w.groups, rows);
    hipLaunchKernelGGL(k_sample_max<VEC>, grid, dim3(LG_T), 0, st, x, ldx, V, s, w);
    hipLaunchKernelGGL(k_sample_mass<VEC>, grid, dim3(LG_T), 0, st, x, ldx, V, s, w, ids, probs);
    if (s.temp && (s.top_k || s.top_p))
        hipLaunchKernelGGL(k_sample_cut<VEC>, grid, dim3(LG_T), 0, st, x, ldx, V, s, w, ids, probs);
}

hipError_t launch_sample(hipStream_t st, const float* x, int64_t ldx, int rows, int V, const SamplingDev& s,
                         int32_t* ids, float* probs, uint8_t* ws) {
    SampleWs w;
    sample_layout(rows, V, ws, w);
    if (vec_rows(x, ldx)) sample_vec<true>(st, x, ldx, rows, V, s, ids, probs, w);
    else sample_vec<false>(st, x, ldx, rows, V, s, ids, probs, w);
    return hipGetLastError();
}
