// Operators on rows of logits in device memory: penalties, biases and grammar
// masks (cc_logits_adjust), and the draw of a token from the adjusted row
// (cc_sample).
#include "common.h"
#include "ops.h"
#include <type_traits>

// ================================================================= adjust ===
// A row's adjusted logits, by chunks of the vocabulary. With c the sum of the
// row's history counts of a token (an entry counts 1 where no counts are
// given):
//   v = x;  c > 0:  v = v > 0 ? v / rep : v * rep;  v -= pres + min(freq * c, cap)
//   + the bias of the token's last entry;  masked out: -inf
// in f64, rounded to f32 once (an untouched token's bits stay as they are).
// An id that occurs twice needs no order: counts add up as integers, and of a
// token's bias entries the largest index wins.
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
    // within the lists whatever the offsets say, both ends: an end past them alone would have the loops' indices wrap
    if (s.pen_at) {
        r.p0 = min(max(s.pen_at[row], 0), s.n_pen);
        r.p1 = min(max(s.pen_at[row + 1], 0), s.n_pen);
    }
    if (s.bias_at) {
        r.b0 = min(max(s.bias_at[row], 0), s.n_bias);
        r.b1 = min(max(s.bias_at[row + 1], 0), s.n_bias);
    }
    r.mask = nullptr;
    if (s.mask) {
        const int m = s.mask_of[row];
        if (m >= 0 && m < s.n_masks) r.mask = s.mask + (size_t)m * s.mask_words;
    }
    return r;
}

constexpr int LG_CH = 4096;

__device__ static inline float adjust_one(float x, const SamplingDev& s, const RowPens& r, uint32_t cnt, int last) {
    if (cnt == 0 && last <= 0) return x;
    double v = (double)x;
    if (cnt != 0) {
        v = v > 0.0 ? v / r.rep : v * r.rep;
        v -= r.pres + fmin(r.freq * (double)cnt, r.cap);
    }
    if (last > 0) v += (double)s.bias[r.b0 + last - 1];
    return (float)v;
}

// A chunk is LG_CH tokens, LG_PER a thread: LG_J runs of four, run j of thread
// t at 4 * (LG_T * j + t). a: the chunk's adjusted logits of row x, in that
// order; -inf past the vocabulary and where the mask bars the token. VEC: the
// row's fours of logits are 16-byte aligned; LISTS: the call has histories or
// biases (without, no LDS holds the workgroups of a CU down); NT: the
// logits pass the caches' ordinary way.
constexpr int LG_J = LG_CH / (4 * LG_T);

// Applies the row's lists to its chunk at `base`. What a token is listed for
// is gathered in LDS first (LG_CH words): its count in the upper half of its
// word, its last bias entry + 1 in the lower. Where those do not fit (a row of
// 2^16 entries, or counts of the caller's), each half of the chunk in turn
// gets a word for either; a count that passes 32 bits stays at 2^32 - 1 (told by
// the top bit of the bias word, which no entry's index reaches).
__device__ static inline void apply_lists(const SamplingDev& s, const RowPens& r, int base, uint32_t* lds,
                                          float (&a)[LG_J][4]) {
    const int tid = threadIdx.x;
    const bool narrow = !s.pen_counts && r.p1 - r.p0 < 65536 && r.b1 - r.b0 < 65535;
    for (int h = 0; h < (narrow ? 1 : 2); h++) {
        const uint32_t first = base + h * (LG_CH / 2), n = narrow ? LG_CH : LG_CH / 2;
        __syncthreads();   // what was here is read
        for (int i = 4 * tid; i < LG_CH; i += 4 * LG_T) *(uint4*)(lds + i) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        for (uint32_t i = r.b0 + tid; i < (uint32_t)r.b1; i += LG_T) {
            const uint32_t at = (uint32_t)s.bias_ids[i] - first;
            if (at < n) atomicMax(&lds[narrow ? at : LG_CH / 2 + at], i - r.b0 + 1);
        }
        if (r.b0 < r.b1) __syncthreads();   // the largest of whole words, before counts and the top bit come in above
        for (uint32_t i = r.p0 + tid; i < (uint32_t)r.p1; i += LG_T) {
            const uint32_t at = (uint32_t)s.pen_ids[i] - first;
            const int c = s.pen_counts ? s.pen_counts[i] : 1;
            if (at >= n || c <= 0) continue;
            if (narrow) atomicAdd(&lds[at], 0x10000u);
            else if (atomicAdd(&lds[at], (uint32_t)c) > 0xffffffffu - (uint32_t)c) atomicOr(&lds[LG_CH / 2 + at], 0x80000000u);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < LG_J; j++) {
            if (!narrow && j / (LG_J / 2) != h) continue;
            const int i = 4 * (LG_T * j + tid) - (narrow ? 0 : h * (LG_CH / 2));
            const uint4 u = *(const uint4*)(lds + i);
            const uint4 l = narrow ? make_uint4(u.x & 0xffffu, u.y & 0xffffu, u.z & 0xffffu, u.w & 0xffffu)
                                   : *(const uint4*)(lds + LG_CH / 2 + i);
            const int up = narrow ? 16 : 0;
            if ((u.x | u.y | u.z | u.w | l.x | l.y | l.z | l.w) != 0) {   // few of the fours hold a listed token
                auto one = [&](float& x, uint32_t cnt, uint32_t last) {
                    x = adjust_one(x, s, r, (int)last < 0 ? 0xffffffffu : cnt >> up, (int)(last & 0x7fffffffu));
                };
                one(a[j][0], u.x, l.x);
                one(a[j][1], u.y, l.y);
                one(a[j][2], u.z, l.z);
                one(a[j][3], u.w, l.w);
            }
        }
    }
}

template <bool VEC, bool LISTS, bool NT = false>
__device__ static inline void adjusted_chunk(const float* __restrict__ x, int V, const SamplingDev& s, const RowPens& r,
                                             int base, uint32_t* lds, float (&a)[LG_J][4]) {
#pragma unroll
    for (int j = 0; j < LG_J; j++) {
        const int t = base + 4 * (LG_T * j + (int)threadIdx.x);
        if (VEC && t + 3 < V) {
            const float4_t f = NT ? __builtin_nontemporal_load((const float4_t*)(x + t)) : *(const float4_t*)(x + t);
            a[j][0] = f[0]; a[j][1] = f[1]; a[j][2] = f[2]; a[j][3] = f[3];
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
    if (LISTS && (r.p0 < r.p1 || r.b0 < r.b1)) apply_lists(s, r, base, lds, a);
#pragma unroll
    for (int j = 0; j < LG_J; j++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (!((bits[j] >> e) & 1u)) a[j][e] = -INFINITY;
}

// What bounds it at many rows is memory. Its loads and stores are non-temporal:
// 128 x 248320 (254 MB in and out), in turn with two other calls' buffers,
// takes 84 us with ordinary ones and 68 with these; up to 64 rows x 151936,
// alone or with the sampler reading its output, the two are the same.
template <bool VEC, bool LISTS>
__global__ __launch_bounds__(LG_T) void k_logits_adjust(const float* x, int64_t ldx, int V, SamplingDev s, float* out,
                                                        int64_t ldo) {
    __shared__ __align__(16) uint32_t lds[LISTS ? LG_CH : 4];
    const int row = blockIdx.y, base = blockIdx.x * LG_CH;
    float a[LG_J][4];
    adjusted_chunk<VEC, LISTS, true>(x + row * ldx, V, s, row_pens(s, row), base, lds, a);
#pragma unroll
    for (int j = 0; j < LG_J; j++) {
        const int t = base + 4 * (LG_T * j + (int)threadIdx.x);
        float* o = out + row * ldo + t;
        if (VEC && t + 3 < V) {
            const float4_t f = {a[j][0], a[j][1], a[j][2], a[j][3]};
            __builtin_nontemporal_store(f, (float4_t*)o);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (t + e < V) o[e] = a[j][e];
        }
    }
}

static bool vec_rows(const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 4 == 0; }
static bool has_lists(const SamplingDev& s) { return s.pen_at || s.bias_at; }
// f with (VEC, LISTS) as types.
template <class F>
static hipError_t with_forms(bool vec, bool lists, F&& f) {
    if (vec && lists) return f(std::true_type{}, std::true_type{});
    if (vec) return f(std::true_type{}, std::false_type{});
    if (lists) return f(std::false_type{}, std::true_type{});
    return f(std::false_type{}, std::false_type{});
}

hipError_t launch_logits_adjust(hipStream_t st, const float* x, int64_t ldx, int rows, int V, const SamplingDev& s,
                                float* out, int64_t ldo) {
    const dim3 grid((V + LG_CH - 1) / LG_CH, rows);
    return with_forms(vec_rows(x, ldx) && vec_rows(out, ldo), has_lists(s), [&](auto vec, auto lists) {
        return op_launch(k_logits_adjust<vec.value, lists.value>, grid, dim3(LG_T), st, x, ldx, V, s, out, ldo);
    });
}

// ================================================================= sample ===
// With a the adjusted row (a NaN counts as -inf) and temp > 0:
//   s = f32(a / temp) (a finite value stays finite), m = max s,
//   w = exp(s - m) as a whole number of 2^-42, so that sums of weights are
//   exact integers and do not depend on their order (a row without cuts: by
//   chunk, relative to the chunk's maximum; the chunks' sums then relative to m
//   and whole numbers again);
//   kept by top-k: s >= the k-th largest s (ties stay);
//   kept by top-p: s >= the largest value t for which the kept weights of
//   s >= t reach p of all kept weights (ties stay);
//   kept by min-p: exp(s - m) >= min_p;
//   token: the first whose running sum of kept weights, in the order of the
//   ids, is above u * sum; prob = exp(s - m) / sum.
// temp <= 0 (or null): the first maximum of a, prob 1. No token left: -1, 0.
//
// Calls without top-k, top-p and min-p take two launches and read the logits
// once:
//   k_sample_weights  the weight of every chunk, relative to its own maximum;
//   k_sample_pick     a workgroup a row: the chunk that the token falls into,
//                     and the token in it.
// The others take three:
//   k_sample_scale    writes s to the workspace, with every chunk's largest and
//                     smallest value: lists, masks and the division once;
//   k_sample_mass     with the row's m known, a histogram of m - s in SM_BINS
//                     bins (counts for top-k, weights for top-p), by chunk
//                     and of the row; the row's last workgroup to finish
//                     finds the bins that the cuts fall into. (A row
//                     with min-p alone: the weights, and the last one draws.)
//   k_sample_cut      the values of those bins are gathered; the row's last
//                     workgroup finds the cuts' exact values among them and
//                     draws. Where everything up to the cut's bin is at most
//                     SM_SMALL values, all of it is gathered, and each value
//                     counts the larger ones; else 9 bits at a time.
// A row of such a call that asks for no cut is drawn as in the other kind, from
// the same whole numbers (k_sample_scale sums its chunks' weights, the first
// workgroup of k_sample_mass picks), so its token and probability do not
// depend on what its neighbours ask for.
// A row with more than SM_CAND values in the bins from its cuts' lowest to their
// highest is drawn by its last workgroup alone, in passes over the row. That is
// where one finite value far below the others widens the bins to 1/16 (a ban of
// -1e4 on logits with a spread of 0.5: 151936 of them with top-p take 1.7 ms
// instead of 0.04, 32 such rows 1.9 instead of 0.06), and where top-k is large
// and top-p cuts far above it (k 20000, p 0.5: 0.7-0.9 ms a row, 32 rows 1.3).
//
// 128 rows of 128256 without cuts: 27 + 8 us, bound by the issue of vector
// instructions: 877 for a lane's 16 logits, a third of them the f64 of the
// weights; the rest follows the first maximum by token, applies masks and keeps
// finite values finite (the logits' bytes alone take 13). 32 rows of 151936 with
// top-p and min-p: 15.7 + 17.7 + 17.8 us, the weights' histogram in LDS, then
// one workgroup a row that finds the cut (3 us) and draws (5). One row of 49152
// with top-k: 7 + 7 + 9 us, a chain of loads and barriers.
constexpr int SM_BINS = 512, SM_CAND = 4096, SM_SMALL = 512, SM_CHUNKS = (1 << 20) / LG_CH;
constexpr float SM_REACH = 32.0f;            // the histogram's last bin takes everything below m - 32
constexpr double SM_ONE = 4398046511104.0;   // 2^42: a row of 2^20 tokens sums to at most 2^62
constexpr double SM_LEAST = 1e-13;           // under half a 2^-42
typedef unsigned long long u64;

// 1 / temp, never 0: a barred token's -inf stays so at an infinite temperature.
__device__ static inline double inverse(double temp) { return temp > 0.0 ? fmax(1.0 / temp, 1e-300) : 1.0; }
// s of an adjusted logit. inv = 1/temp; only above 1 can a finite value leave
// the range (a branch on it is uniform).
__device__ static inline float scaled_logit(float a, double inv) {
    a = fmaxf(a, -INFINITY);   // NaN: -inf
    float s = (float)((double)a * inv);
    if (inv > 1.0 && fabsf(a) < INFINITY) s = fminf(fmaxf(s, -3.4028234663852886e38f), 3.4028234663852886e38f);
    return s + 0.0f;   // -0 is 0
}

// 2^(j/32), j = 0 .. 31, in LDS: 256 bytes, so a lane's lookup meets no bank
// conflict.
__device__ static inline void exp_table(double* T) {
    static constexpr double two32[32] = {
        1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924,
        1.1387886347566916, 1.1637248587775775, 1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
        1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832, 1.4142135623730951, 1.4451808069770467,
        1.4768261459394993, 1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.6457554781539649,
        1.681792830507429, 1.7186192981224779, 1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103,
        1.9152065613971474, 1.9571441241754002};
    if (threadIdx.x < 32) T[threadIdx.x] = two32[threadIdx.x];
}
// exp(s - m) in [0, 1], s <= m, in pieces: x = (32 e + j) ln2/32 + r with |r| <=
// ln2/64, exp(r) to five terms (left off: r^6/720 < 2^-48) and 2^e * 2^(j/32)
// with the exponent put into the table's entry. Under x = -30 the weight is
// less than half a 2^-42 and counts as nothing. (fmin also takes inf - inf,
// a NaN, to 0: the weight of +inf is 1.)
struct ExpParts {
    double p, t;
    bool some;
};
__device__ static inline ExpParts exp_parts(float s, double m, const double* T) {
    const double x = fmin((double)s - m, 0.0);
    const double n = rint(x * 46.16624130844683);   // 32 / ln 2
    const int i = (int)n;
    const double r = fma(n, -0.02166084939249829, x);
    double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const u64 b = __builtin_bit_cast(u64, T[i & 31]);
    const uint32_t hi = (uint32_t)(b >> 32) + ((uint32_t)(i >> 5) << 20);
    return ExpParts{p, __builtin_bit_cast(double, (u64)hi << 32 | (uint32_t)b), x > -30.0};
}
__device__ static inline double weight(float s, float m, const double* T) {
    const ExpParts e = exp_parts(s, (double)m, T);
    return e.some ? e.p * e.t : 0.0;
}
// The weight to the nearest 2^-42, as a whole number above SM_BASE: 2^10 + w
// has that step.
constexpr u64 SM_BASE = 0x4090000000000000ull;   // the bits of 1024.0
__device__ static inline u64 based_weight(float s, double m, const double* T) {
    const ExpParts e = exp_parts(s, m, T);
    return e.some ? __builtin_bit_cast(u64, fma(e.p, e.t, 1024.0)) : SM_BASE;
}
__device__ static inline u64 whole_weight(float s, float m, const double* T) { return based_weight(s, (double)m, T) - SM_BASE; }

__device__ static inline uint32_t ordered(float v) {
    const uint32_t b = f2u(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ static inline float unordered(uint32_t k) { return u2f((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

// min-p as a cut of s: the ordered bits of the smallest value whose weight
// reaches min_p (0: none is cut; a weight under SM_LEAST counts as nothing anyhow).
// Mostly m + log(min_p) to a step; but next to zero an f32 step is so short
// that millions of values share a weight (min_p 1 and m 0: all of the 10^9 from
// -2^-54 up weigh 1), so the search's steps double and then halve: 64 at most.
__device__ static inline uint32_t min_cut(float m, double min_p, const double* T) {
    if (!(min_p > SM_LEAST)) return 0;
    if (m == INFINITY) return ordered(m);
    const uint32_t top = ordered(m), least = ordered((float)((double)m - 31.0)) - 1;   // it weighs nothing
    auto cut = [&](uint32_t k) { return k <= least || (k < top && weight(unordered(k), m, T) < min_p); };
    uint32_t lo = ordered(fminf((float)((double)m + log(min_p)), m)), hi = lo;
    for (uint32_t step = 1; cut(hi); step *= 2) {
        lo = hi;
        hi = step < top - hi ? hi + step : top;
    }
    for (uint32_t step = 1; !cut(lo); step *= 2) {
        hi = lo;
        lo = step < lo - least ? lo - step : least;
    }
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (cut(mid)) lo = mid;
        else hi = mid;
    }
    return hi;
}

// A lane's 64-bit value from another lane by DPP (zero where there is none).
template <int CTRL, int ROWS = 0xf>
__device__ static inline u64 dpp64(u64 v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
    return (u64)hi << 32 | lo;
}
__device__ static inline u64 lane64(u64 v, int lane) {
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
// The sum over a wave's lanes up to this one: within rows of 16 lanes by
// shifts (1, 2, 4, 8), then the rows' sums before.
__device__ static inline u64 wave_scan64(u64 v) {
    v += dpp64<0x111>(v);
    v += dpp64<0x112>(v);
    v += dpp64<0x114>(v);
    v += dpp64<0x118>(v);
    const u64 a = lane64(v, 15), b = a + lane64(v, 31), c = b + lane64(v, 47);
    const int row = (threadIdx.x & 63) >> 4;
    return v + (row == 0 ? 0 : row == 1 ? a : row == 2 ? b : c);
}
__device__ static inline u64 wave_max64(u64 v) {
    auto mx = [](u64 a, u64 b) { return a > b ? a : b; };
    v = mx(v, dpp64<0xB1>(v));
    v = mx(v, dpp64<0x4E>(v));
    v = mx(v, dpp64<0x141>(v));
    v = mx(v, dpp64<0x140>(v));
    return mx(mx(lane64(v, 0), lane64(v, 16)), mx(lane64(v, 32), lane64(v, 48)));
}
// Over the workgroup, to every thread: the sum; the sum of the threads before
// (red then holds the waves' sums); the largest.
__device__ static inline u64 block_before64(u64 v, u64* red) {
    u64 inc = wave_scan64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = inc;
    __syncthreads();
    for (int w = 0; w < (int)(threadIdx.x >> 6); w++) inc += red[w];
    return inc - v;
}
__device__ static inline u64 block_sum64(u64 v, u64* red) {
    block_before64(v, red);
    return red[0] + red[1] + red[2] + red[3];
}
__device__ static inline u64 block_max64(u64 v, u64* red) {
    v = wave_max64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    const u64 a = red[0] > red[1] ? red[0] : red[1], b = red[2] > red[3] ? red[2] : red[3];
    return a > b ? a : b;
}

// The workspace of a call: per row and chunk the largest key and the weight;
// with cuts also the smallest value and the weights' histogram, and per row the
// histograms, the scaled logits, what the cuts found, two counters of finished
// workgroups and the gathered values.
struct SampleInfo {
    int32_t lo, hi;        // the bins whose values are gathered
    uint32_t above;        // values in the bins before lo
    uint32_t n_cand;       // gathered values (more than SM_CAND: not all of them were)
    u64 mass_above;        // the weight of the bins before lo
    u64 want;              // top-p without top-k: the weight to reach
    uint32_t floor, fixed; // min-p as a value's ordered bits; whether it is the cut
    uint32_t done[2];
    float m, bins;         // RowDraw's (bins 0: no cut to find)
};
struct SampleWs {
    u64* best;        // [rows][chunks] ordered(a) << 32 | ~token; 0: nothing above -inf
    float* least;     // [rows][chunks] the smallest value above -inf
    u64* mass;        // [rows][chunks]
    u64* hmass;       // [rows][chunks][SM_BINS]
    u64* rmass;       // [rows][SM_BINS] the chunks' sums
    uint32_t* rcount; // [rows][SM_BINS] values in them
    SampleInfo* info; // [rows]
    uint2* cand;      // [rows][SM_CAND] ordered(s), token
    float* s;         // [rows][lds]
    int64_t lds;
    int chunks;
};

struct RowAsk {
    double inv, top_p, min_p;
    bool greedy, cut, plain;   // cut: by top-k or top-p; plain: by nothing
    int k;
    __device__ RowAsk(const SamplingDev& s, int row, int V) {
        const double temp = s.temp ? (double)s.temp[row] : 0.0;
        greedy = !(temp > 0.0);
        inv = inverse(temp);
        k = s.top_k ? s.top_k[row] : 0;
        if (k >= V || k < 0) k = 0;
        top_p = s.top_p ? (double)s.top_p[row] : 1.0;
        if (!(top_p < 1.0)) top_p = 1.0;
        min_p = s.min_p ? (double)s.min_p[row] : 0.0;
        if (min_p > 1.0) min_p = 1.0;   // the maximum itself stays
        cut = !greedy && (k > 0 || top_p < 1.0);
        plain = !greedy && !cut && !(min_p > SM_LEAST);
    }
};

__device__ static inline u64 best_key(float a, uint32_t token) {
    return a > -INFINITY ? (u64)ordered(a + 0.0f) << 32 | (0xffffffffu - token) : 0;   // -0 is 0
}
// The first largest of values given in the order of their tokens (-0 is 0, a
// NaN nothing).
struct FirstMax {
    float v = -INFINITY;
    uint32_t t = 0;
    __device__ void take(float a, uint32_t token) {
        const bool more = a > v;
        v = more ? a : v;
        t = more ? token : t;
    }
    __device__ u64 key() const { return best_key(v, t); }
};
__device__ static inline u64 target_of(double u, u64 total) {
    const u64 t = (u64)fmax(u * (double)total, 0.0);
    return t < total - 1 ? t : total - 1;
}

// Of the scaled logits v of N runs of 4 * LG_T tokens (a chunk's are LG_J, in
// adjusted_chunk's order), the token with `left` of their kept weights before
// it. Called by the whole workgroup; mw(v) is a value's kept weight;
// hit(token, v) is called once. runs: LDS for the runs' weights by wave.
template <int N, class W, class H>
__device__ static inline void draw_in_runs(const float (&v)[N][4], int base, u64 left, u64 (&runs)[N][4], W&& mw, H&& hit) {
    const int wave = threadIdx.x >> 6;
    u64 m[N][4], inc[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        u64 sum = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            m[j][e] = mw(v[j][e]);
            sum += m[j][e];
        }
        inc[j] = wave_scan64(sum);
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63)
#pragma unroll
        for (int j = 0; j < N; j++) runs[j][wave] = inc[j];
    __syncthreads();
    u64 ahead = 0;   // of the weights, before the run and wave
    bool found = false;
#pragma unroll
    for (int j = 0; j < N; j++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const u64 here = runs[j][q];
            if (!found && left < ahead + here) {   // the same for every thread
                found = true;
                if (q == wave) {
                    u64 before = ahead + inc[j] - (m[j][0] + m[j][1] + m[j][2] + m[j][3]);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if (before <= left && left < before + m[j][e]) hit(base + 4 * (LG_T * j + (int)threadIdx.x) + e, v[j][e]);
                        before += m[j][e];
                    }
                }
            }
            ahead += here;
        }
}

// ---- without cuts
// The weight of a chunk of adjusted logits relative to its own maximum (best),
// to every thread.
__device__ static inline u64 chunk_weight(const float (&a)[LG_J][4], u64 best, double inv, const double* T, u64* red) {
    const float m = scaled_logit(unordered((uint32_t)(best >> 32)), inv);
    u64 sum = 0;
#pragma unroll
    for (int j = 0; j < LG_J; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) sum += based_weight(scaled_logit(a[j][e], inv), (double)m, T);
    return block_sum64(sum - LG_J * 4 * SM_BASE, red);
}

// The token of a row, from its chunks' maxima and weights (mine and local:
// those of chunk threadIdx.x; key: the row's best). The chunks' weights
// relative to the row's maximum m are theirs times exp(m_c - m), rounded to
// whole numbers again. load(c, v): the scaled logits of chunk c.
template <class L>
__device__ static inline void pick_row(u64 key, u64 mine, u64 local, double inv, double u, const double* T, u64* red, u64* found,
                                       float* s_m, u64 (&runs)[LG_J][4], int32_t* id, float* prob, L&& load) {
    const float m = scaled_logit(unordered((uint32_t)(key >> 32)), inv);
    const float mc = mine ? scaled_logit(unordered((uint32_t)(mine >> 32)), inv) : -INFINITY;
    const double f = weight(mc, m, T);
    const u64 mass = (u64)rint((double)local * f);
    const u64 before = block_before64(mass, red);
    const u64 total = red[0] + red[1] + red[2] + red[3];
    const u64 target = target_of(u, total);
    if (before <= target && target < before + mass) {
        const u64 left = (u64)((double)(target - before) / f);
        found[0] = threadIdx.x;
        found[1] = left < local - 1 ? left : local - 1;
        *s_m = mc;
    }
    __syncthreads();
    const int c = (int)found[0];
    const u64 left = found[1];
    const float m_c = *s_m;
    float v[LG_J][4];
    load(c, v);
    draw_in_runs(v, c * LG_CH, left, runs, [&](float x) { return whole_weight(x, m_c, T); }, [&](int t, float x) {
        *id = t;
        if (prob) *prob = (float)(weight(x, m, T) * SM_ONE / (double)total);
    });
}

template <bool VEC, bool LISTS>
__global__ __launch_bounds__(LG_T) void k_sample_weights(const float* __restrict__ x, int64_t ldx, int V, SamplingDev s,
                                                         SampleWs w) {
    __shared__ __align__(16) uint32_t lds[LISTS ? LG_CH : 4];
    __shared__ double T[32];
    __shared__ u64 red[4];
    const int row = blockIdx.y, c = blockIdx.x;
    exp_table(T);
    const double temp = s.temp ? (double)s.temp[row] : 0.0, inv = inverse(temp);
    float a[LG_J][4];
    adjusted_chunk<VEC, LISTS>(x + row * ldx, V, s, row_pens(s, row), c * LG_CH, lds, a);
    FirstMax first;
#pragma unroll
    for (int j = 0; j < LG_J; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) first.take(a[j][e], c * LG_CH + 4 * (LG_T * j + threadIdx.x) + e);
    const u64 best = block_max64(first.key(), red);
    const u64 sum = best && temp > 0.0 ? chunk_weight(a, best, inv, T, red) : 0;
    if (threadIdx.x == 0) {
        w.best[(size_t)row * w.chunks + c] = best;
        w.mass[(size_t)row * w.chunks + c] = sum;
    }
}

template <bool VEC, bool LISTS>
__global__ __launch_bounds__(LG_T) void k_sample_pick(const float* __restrict__ x, int64_t ldx, int V, SamplingDev s,
                                                      SampleWs w, int32_t* __restrict__ ids, float* __restrict__ probs) {
    __shared__ __align__(16) uint32_t lds[LISTS ? LG_CH : 4];
    __shared__ double T[32];
    __shared__ u64 red[4], found[2], runs[LG_J][4];
    __shared__ float s_m;
    const int row = blockIdx.x, tid = threadIdx.x;
    exp_table(T);
    const double temp = s.temp ? (double)s.temp[row] : 0.0, inv = inverse(temp);
    const u64 mine = tid < w.chunks ? w.best[(size_t)row * w.chunks + tid] : 0;
    const u64 local = tid < w.chunks ? w.mass[(size_t)row * w.chunks + tid] : 0;
    const u64 key = block_max64(mine, red);
    if (!key || !(temp > 0.0)) {
        if (tid == 0) {
            ids[row] = key ? (int32_t)(0xffffffffu - (uint32_t)key) : -1;
            if (probs) probs[row] = key ? 1.0f : 0.0f;
        }
        return;
    }
    pick_row(key, mine, local, inv, s.u ? s.u[row] : 0.0, T, red, found, &s_m, runs, ids + row, probs ? probs + row : nullptr,
             [&](int c, float (&v)[LG_J][4]) {
                 adjusted_chunk<VEC, LISTS>(x + row * ldx, V, s, row_pens(s, row), c * LG_CH, lds, v);
#pragma unroll
                 for (int j = 0; j < LG_J; j++)
#pragma unroll
                     for (int e = 0; e < 4; e++) v[j][e] = scaled_logit(v[j][e], inv);
             });
}

// ---- with cuts
template <bool VEC, bool LISTS>
__global__ __launch_bounds__(LG_T) void k_sample_scale(const float* __restrict__ x, int64_t ldx, int V, SamplingDev s,
                                                       SampleWs w) {
    __shared__ __align__(16) uint32_t lds[LISTS ? LG_CH : 4];
    __shared__ double T[32];
    __shared__ u64 red[4];
    const int row = blockIdx.y, c = blockIdx.x;
    exp_table(T);
    if (c == 0) {   // the next launch adds to them
        if (threadIdx.x < sizeof(SampleInfo) / 4) ((uint32_t*)(w.info + row))[threadIdx.x] = 0;
        for (int b = threadIdx.x; b < SM_BINS; b += LG_T) {
            w.rmass[(size_t)row * SM_BINS + b] = 0;
            w.rcount[(size_t)row * SM_BINS + b] = 0;
        }
    }
    const RowPens r = row_pens(s, row);
    const RowAsk ask(s, row, V);
    const double inv = ask.inv;
    FirstMax first;
    float least = INFINITY, a[LG_J][4];
    adjusted_chunk<VEC, LISTS>(x + row * ldx, V, s, r, c * LG_CH, lds, a);
#pragma unroll
    for (int j = 0; j < LG_J; j++) {
        const int t = c * LG_CH + 4 * (LG_T * j + (int)threadIdx.x);
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            first.take(a[j][e], t + e);
            least = a[j][e] > -INFINITY ? fminf(least, a[j][e]) : least;
            v[e] = scaled_logit(a[j][e], inv);
        }
        // past the caches' ordinary way: 1.5% of the call less than plain stores, which the kernel's end writes back
        if (t < V) __builtin_nontemporal_store(float4_t{v[0], v[1], v[2], v[3]}, (float4_t*)(w.s + row * w.lds + t));
    }
    const u64 best = block_max64(first.key(), red);
    const u64 low = block_max64(~(u64)ordered(least), red);
    if (threadIdx.x == 0) {
        w.best[(size_t)row * w.chunks + c] = best;
        w.least[(size_t)row * w.chunks + c] = unordered((uint32_t)~low);
    }
    if (!ask.plain) return;
    const u64 sum = best ? chunk_weight(a, best, inv, T, red) : 0;
    if (threadIdx.x == 0) w.mass[(size_t)row * w.chunks + c] = sum;
}

// N runs of a row's scaled logits, from token `base` on.
template <int N>
__device__ static inline void scaled_runs(const float* __restrict__ s, int V, int base, float (&v)[N][4]) {
#pragma unroll
    for (int j = 0; j < N; j++) {
        const int t = base + 4 * (LG_T * j + (int)threadIdx.x);
        const float4 f = t < V ? *(const float4*)(s + t) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        v[j][0] = f.x; v[j][1] = f.y; v[j][2] = f.z; v[j][3] = f.w;
    }
}

// What a row's workgroups share about its draw.
struct RowDraw {
    float m, bins;      // the largest s; bins per unit of m - s
    u64 key;            // the row's best (k_sample_scale)
};
__device__ static inline RowDraw row_draw(const SampleWs& w, int row, const RowAsk& ask, u64* red) {
    u64 best = 0, low = 0;
    for (int i = threadIdx.x; i < w.chunks; i += LG_T) {
        const u64 b = w.best[(size_t)row * w.chunks + i];
        best = b > best ? b : best;
        const u64 l = ~(u64)ordered(w.least[(size_t)row * w.chunks + i]);
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

// The last workgroup of a row, with the workgroups' kept weights known: mass
// (this thread's workgroup of the row) -> the token.
template <int N, class W>
__device__ static inline void draw_row(const float* __restrict__ sr, int V, const SamplingDev& s, int row, u64 mass, float m,
                                       const double* T, u64* red, u64* found, u64 (&runs)[N][4], W&& mw, int32_t* id,
                                       float* prob) {
    const u64 before = block_before64(mass, red);
    const u64 total = red[0] + red[1] + red[2] + red[3];
    const u64 target = target_of(s.u ? s.u[row] : 0.0, total);
    __syncthreads();
    if (before <= target && target < before + mass) {
        found[0] = threadIdx.x;
        found[1] = target - before;
    }
    __syncthreads();
    const int base = (int)found[0] * (N * 4 * LG_T);
    float v[N][4];
    scaled_runs(sr, V, base, v);
    draw_in_runs(v, base, found[1], runs, mw, [&](int t, float q) {
        *id = t;
        if (prob) *prob = (float)(weight(q, m, T) * SM_ONE / (double)total);
    });
}

__global__ __launch_bounds__(LG_T) void k_sample_mass(int V, SamplingDev s, SampleWs w, int32_t* __restrict__ ids,
                                                      float* __restrict__ probs) {
    __shared__ u64 hmass[SM_BINS], red[4], found[2], runs[LG_J][4];
    __shared__ uint32_t hcount[SM_BINS], s_last;
    __shared__ double T[32];
    __shared__ float s_m;
    const int row = blockIdx.y, g = blockIdx.x, tid = threadIdx.x;
    const float* sr = w.s + row * w.lds;
    float v[LG_J][4];
    scaled_runs(sr, V, g * LG_CH, v);   // in flight while the row's maximum is found
    exp_table(T);
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
    if (ask.plain) {   // as in a call without cuts, from the scaled logits
        if (g != 0) return;
        const bool on = tid < w.chunks;
        pick_row(d.key, on ? w.best[(size_t)row * w.chunks + tid] : 0, on ? w.mass[(size_t)row * w.chunks + tid] : 0, ask.inv,
                 s.u ? s.u[row] : 0.0, T, red, found, &s_m, runs, ids + row, prob,
                 [&](int c, float (&x)[LG_J][4]) { scaled_runs(sr, V, c * LG_CH, x); });
        return;
    }
    SampleInfo* info = w.info + row;
    const size_t at = (size_t)row * w.chunks + g;
    if (!ask.cut) {
        const uint32_t cut = min_cut(d.m, ask.min_p, T);
        auto mw = [&](float v) { return ordered(v) >= cut ? whole_weight(v, d.m, T) : 0; };
        u64 sum = 0;
#pragma unroll
        for (int j = 0; j < LG_J; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) sum += mw(v[j][e]);
        sum = block_sum64(sum, red);
        if (tid == 0) leave64(&w.mass[at], sum);
        if (!finished_last(&info->done[0], w.chunks, &s_last)) return;
        draw_row(sr, V, s, row, tid < w.chunks ? left64(&w.mass[(size_t)row * w.chunks + tid]) : 0, d.m, T, red, found, runs, mw,
                 ids + row, prob);
        return;
    }
    // the histogram: counts for top-k, weights for top-p
    const bool weigh = ask.top_p < 1.0, count = ask.k > 0 || !weigh;
    for (int b = tid; b < SM_BINS; b += LG_T) {
        hmass[b] = 0;
        hcount[b] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < LG_J; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (!(v[j][e] > -INFINITY)) continue;
            const int b = bin_of(v[j][e], d);
            if (count) atomicAdd(&hcount[b], 1u);
            if (weigh) atomicAdd(&hmass[b], whole_weight(v[j][e], d.m, T));
        }
    __syncthreads();
    // the row's sums by atomics on whole numbers, whose order does not matter (32 rows of 38 workgroups: 3.3 us less than
    // with the last one reading all the histograms); the weights also by workgroup, for the next launch
    auto add = [](auto* p, auto v) {
        if (v) __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    for (int b = tid; b < SM_BINS; b += LG_T) {
        if (count) add(&w.rcount[(size_t)row * SM_BINS + b], hcount[b]);
        if (weigh) {
            w.hmass[at * SM_BINS + b] = hmass[b];
            add(&w.rmass[(size_t)row * SM_BINS + b], hmass[b]);
        }
    }
    if (!finished_last(&info->done[0], w.chunks, &s_last)) return;
    // thread t: bins 2t and 2t + 1
    const size_t mine = (size_t)row * SM_BINS + 2 * tid;
    const u64 c2 = count ? left64(&w.rcount[mine]) : 0;
    const u64 n[2] = {c2 & 0xffffffffu, c2 >> 32};
    const u64 ms[2] = {weigh ? left64(&w.rmass[mine]) : 0, weigh ? left64(&w.rmass[mine + 1]) : 0};
    const u64 nb = block_before64(n[0] + n[1], red);
    const u64 mb = block_before64(ms[0] + ms[1], red);
    const u64 total = red[0] + red[1] + red[2] + red[3];
    // the bin in which a running sum (of counts or weights) first reaches `want`
    auto reach = [&](u64 before, const u64* v, u64 want) {
        __syncthreads();
        if (tid == 0) found[0] = SM_BINS - 1;
        __syncthreads();
        if (before < want && want <= before + v[0] + v[1]) found[0] = 2 * tid + (before + v[0] < want ? 1 : 0);
        __syncthreads();
        return (int)found[0];
    };
    // a sum over the bins before b
    auto ahead = [&](u64 before, const u64* v, int b) {
        __syncthreads();
        if (tid == b >> 1) found[0] = before + ((b & 1) ? v[0] : 0);
        __syncthreads();
        return found[0];
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
    // few enough up to and with hi: all of them are gathered
    if (count && hi + 1 < SM_BINS && ahead(nb, n, hi + 1) <= SM_SMALL) lo = 0;
    // min-p cuts above what top-k and top-p cut: only its own bin is looked at
    const uint32_t floor = min_cut(d.m, ask.min_p, T);
    const int fb = floor ? bin_of(unordered(floor), d) : SM_BINS;
    const bool fixed = fb < lo;
    if (fixed) lo = hi = fb;
    const u64 above = ahead(nb, n, lo), mass_above = weigh ? ahead(mb, ms, lo) : 0;
    if (tid == 0) {
        info->lo = lo;
        info->hi = hi;
        info->floor = floor;
        info->fixed = fixed;
        info->above = (uint32_t)above;
        info->mass_above = mass_above;
        info->want = want;
        info->m = d.m;
        info->bins = d.bins;
    }
}

// The value (as ordered bits) at which the sum over the values from the top
// first reaches `want`, 9 bits at a time below the bits that all keys (in
// [kmin, kmax]) share: `each` calls its argument for every value with its key
// and what it adds. kmin (everything is kept) if they all sum to less.
template <class E>
__device__ static inline uint32_t find_cut(u64 want, uint32_t kmin, uint32_t kmax, u64* hist, u64* sel, E&& each) {
    const int tid = threadIdx.x, lane = tid & 63;
    uint32_t prefix = 0;   // of key - kmin
    u64 left = want;
    const int bits = kmax > kmin ? 32 - __clz(kmax - kmin) : 0;
    for (int sh = (bits + 8) / 9 * 9 - 9; sh >= 0; sh -= 9) {
        __syncthreads();
        hist[tid] = 0;
        hist[LG_T + tid] = 0;
        if (tid == 0) {
            sel[0] = prefix;
            sel[1] = left;
        }
        __syncthreads();
        each([&](uint32_t key, u64 adds) {
            const uint32_t k = key - kmin;
            if (sh == 27 || (k >> (sh + 9)) == (prefix >> (sh + 9))) atomicAdd(&hist[(k >> sh) & 511u], adds);
        });
        __syncthreads();
        if (tid < 64) {   // lane l: digits 511 - 8l .. 504 - 8l
            u64 v[8], sum = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[e] = hist[511 - 8 * lane - e];
                sum += v[e];
            }
            u64 before = wave_scan64(sum) - sum;
            if (before < left && left <= before + sum) {
                int e = 0;
#pragma unroll
                for (int q = 0; q < 7; q++)   // no index at run time: the array stays in registers
                    if (e == q && before + v[q] < left) {
                        before += v[q];
                        e = q + 1;
                    }
                sel[0] = prefix | ((uint32_t)(511 - 8 * lane - e) << sh);
                sel[1] = left - before;
            }
        }
        __syncthreads();
        prefix = (uint32_t)sel[0];
        left = sel[1];
    }
    return kmin + prefix;
}

__global__ __launch_bounds__(LG_T) void k_sample_cut(int V, SamplingDev s, SampleWs w, int32_t* __restrict__ ids,
                                                     float* __restrict__ probs) {
    __shared__ __align__(16) uint32_t keys[SM_CAND];
    __shared__ uint8_t group[SM_CAND];   // the chunk that a value came from
    __shared__ __align__(16) u64 wts[SM_SMALL], gmass[LG_T], hist[2 * LG_T], red[4], found[2], runs[LG_J][4];
    __shared__ __align__(16) uint32_t tok[SM_SMALL];
    __shared__ uint32_t s_last, s_n, s_at;
    __shared__ double T[32];
    static_assert(SM_CHUNKS <= LG_T, "a thread a workgroup of the row");
    static_assert(SM_SMALL == 2 * LG_T, "two values a thread");
    const int row = blockIdx.y, g = blockIdx.x, tid = threadIdx.x;
    const RowAsk ask(s, row, V);
    if (!ask.cut) return;
    const float* sr = w.s + row * w.lds;
    float v[LG_J][4];
    scaled_runs(sr, V, g * LG_CH, v);
    exp_table(T);
    SampleInfo* info = w.info + row;
    const RowDraw d{info->m, info->bins, 0};
    if (d.bins == 0.0f) return;
    const int lo = info->lo, hi = info->hi;
    uint2* cand = w.cand + (size_t)row * SM_CAND;
    const uint32_t floor = info->floor;
    const bool from_hist = ask.top_p < 1.0;   // the weights of the bins before lo, all above min-p's, are in the histogram
    if (tid == 0) s_n = 0;
    __syncthreads();   // T is there for every wave, and s_n
    u64 sum = 0;
    if (from_hist) {
        const u64* h = w.hmass + ((size_t)row * w.chunks + g) * SM_BINS;
        for (int b = tid; b < lo; b += LG_T) sum += h[b];
    }
    uint32_t in = 0;
#pragma unroll
    for (int j = 0; j < LG_J; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float q = v[j][e];
            const int b = q > -INFINITY ? bin_of(q, d) : SM_BINS;
            if (b >= lo && b <= hi) in |= 1u << (4 * j + e);
            if (b < lo && !from_hist) sum += whole_weight(q, d.m, T);
        }
    // the workgroup's place among the gathered values, then each thread's
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
                    leave64(&cand[mine], (u64)(g * LG_CH + 4 * (LG_T * j + tid) + e) << 32 | ordered(v[j][e]));
                mine++;
            }
    sum = block_sum64(sum, red);
    if (tid == 0) leave64(&w.mass[(size_t)row * w.chunks + g], sum);
    if (!finished_last(&info->done[1], w.chunks, &s_last)) return;
    const uint32_t n = left32(&info->n_cand);
    const u64 above = info->above, mass_above = info->mass_above;
    auto weigh_key = [&](uint32_t key) { return whole_weight(unordered(key), d.m, T); };
    float* prob = probs ? probs + row : nullptr;
    if (lo == 0 && n <= SM_SMALL && !info->fixed) {
        // every value that may be kept is here, two a thread: it is kept if fewer than k are larger, if the larger ones
        // that top-k keeps have not reached p of the weight, and if it reaches min_p
        uint32_t kv[2];
        u64 mv[2];
        bool in[2];
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const uint32_t i = tid + q * LG_T;
            const u64 c2 = i < n ? left64(&cand[i]) : 0;
            keys[i] = kv[q] = (uint32_t)c2;      // 0: no value has these bits (-inf is left out)
            tok[i] = (uint32_t)(c2 >> 32);
            mv[q] = i < n ? weigh_key(kv[q]) : 0;
            wts[i] = mv[q];
            in[q] = i < n;
        }
        __syncthreads();
        if (ask.k > 0) {
            uint32_t larger[2] = {0, 0};
            for (uint32_t i = 0; i < n; i += 8)   // past n: zeros
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    larger[0] += keys[i + e] > kv[0];
                    larger[1] += keys[i + e] > kv[1];
                }
            in[0] = in[0] && larger[0] < (uint32_t)ask.k;
            in[1] = in[1] && larger[1] < (uint32_t)ask.k;
        }
        if (ask.top_p < 1.0) {
            __syncthreads();
#pragma unroll
            for (int q = 0; q < 2; q++)
                if (!in[q]) wts[tid + q * LG_T] = 0;
            u64 want = info->want;
            if (ask.k > 0)
                want = (u64)fmax(ceil(ask.top_p * (double)block_sum64((in[0] ? mv[0] : 0) + (in[1] ? mv[1] : 0), red)), 1.0);
            __syncthreads();
            u64 over[2] = {0, 0};
            for (uint32_t i = 0; i < n; i += 8)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const u64 x = wts[i + e];
                    const uint32_t kk = keys[i + e];
                    over[0] += kk > kv[0] ? x : 0;
                    over[1] += kk > kv[1] ? x : 0;
                }
            in[0] = in[0] && over[0] < want;
            in[1] = in[1] && over[1] < want;
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 2; q++) {
            if (!in[q] || kv[q] < floor) mv[q] = 0;
            wts[tid + q * LG_T] = mv[q];
        }
        const u64 total = block_sum64(mv[0] + mv[1], red);
        __syncthreads();
        const u64 target = target_of(s.u ? s.u[row] : 0.0, total);
        u64 before[2] = {0, 0};
        const uint32_t t0 = tok[tid], t1 = tok[tid + LG_T];
        for (uint32_t i = 0; i < n; i += 8)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const u64 x = wts[i + e];
                const uint32_t tt = tok[i + e];
                before[0] += tt < t0 ? x : 0;
                before[1] += tt < t1 ? x : 0;
            }
#pragma unroll
        for (int q = 0; q < 2; q++)
            if (before[q] <= target && target < before[q] + mv[q]) {
                ids[row] = (int32_t)(q ? t1 : t0);
                if (prob) *prob = (float)(weight(unordered(kv[q]), d.m, T) * SM_ONE / (double)total);
            }
        return;
    }
    uint32_t cut = 0;
    const bool k_cuts = ask.k > 0 && !info->fixed, p_cuts = ask.top_p < 1.0 && !info->fixed;
    gmass[tid] = tid < w.chunks ? left64(&w.mass[(size_t)row * w.chunks + tid]) : 0;
    if (n <= SM_CAND) {
        u64 top = 0, low = 0;
        for (uint32_t i0 = tid; i0 < n; i0 += 8 * LG_T) {   // eight loads in flight
            u64 q[8];
#pragma unroll
            for (int e = 0; e < 8; e++) q[e] = i0 + e * LG_T < n ? left64(&cand[i0 + e * LG_T]) : 0;
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (i0 + e * LG_T < n) {
                    const uint32_t key = (uint32_t)q[e];
                    keys[i0 + e * LG_T] = key;
                    group[i0 + e * LG_T] = (uint8_t)((uint32_t)(q[e] >> 32) / (uint32_t)LG_CH);
                    top = key > top ? key : top;
                    low = (u64)(~key) > low ? (u64)(~key) : low;
                }
        }
        const uint32_t kmax = (uint32_t)block_max64(top, red), kmin = n ? ~(uint32_t)block_max64(low, red) : 0u;   // none: no cut
        if (k_cuts)
            cut = find_cut((u64)ask.k - above, kmin, kmax, hist, found, [&](auto&& f) {
                for (uint32_t i = tid; i < n; i += LG_T) f(keys[i], 1ull);
            });
        if (p_cuts) {
            u64 want = info->want;
            if (ask.k > 0) {
                u64 in = 0;
                for (uint32_t i = tid; i < n; i += LG_T)
                    if (keys[i] >= cut) in += weigh_key(keys[i]);
                want = (u64)fmax(ceil(ask.top_p * (double)(mass_above + block_sum64(in, red))), 1.0);
            }
            const uint32_t from = cut;
            const uint32_t c2 = find_cut(want - mass_above, kmin, kmax, hist, found, [&](auto&& f) {
                for (uint32_t i = tid; i < n; i += LG_T)
                    if (keys[i] >= from) f(keys[i], weigh_key(keys[i]));
            });
            cut = c2 > cut ? c2 : cut;
        }
        cut = cut > floor ? cut : floor;
        __syncthreads();
        for (uint32_t i = tid; i < n; i += LG_T)
            if (keys[i] >= cut) atomicAdd(&gmass[group[i]], weigh_key(keys[i]));
    } else {
        // too many values share the cut's bins: the same, in passes over the row
        const int chunks = (V + LG_CH - 1) / LG_CH;
        auto all = [&](auto&& f) {
            for (int c = 0; c < chunks; c++) {
                float x[LG_J][4];
                scaled_runs(sr, V, c * LG_CH, x);
#pragma unroll
                for (int j = 0; j < LG_J; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (x[j][e] > -INFINITY) f(ordered(x[j][e]), c);
            }
        };
        if (k_cuts)
            cut = find_cut((u64)ask.k, 0, 0xffffffffu, hist, found, [&](auto&& f) { all([&](uint32_t key, int) { f(key, 1ull); }); });
        if (p_cuts) {
            u64 in = 0;
            all([&](uint32_t key, int) {
                if (key >= cut) in += weigh_key(key);
            });
            const u64 want = (u64)fmax(ceil(ask.top_p * (double)block_sum64(in, red)), 1.0);
            const uint32_t from = cut;
            const uint32_t c2 = find_cut(want, 0, 0xffffffffu, hist, found, [&](auto&& f) {
                all([&](uint32_t key, int) {
                    if (key >= from) f(key, weigh_key(key));
                });
            });
            cut = c2 > cut ? c2 : cut;
        }
        cut = cut > floor ? cut : floor;
        __syncthreads();
        gmass[tid] = 0;
        __syncthreads();
        all([&](uint32_t key, int c) {
            if (key >= cut) atomicAdd(&gmass[c], weigh_key(key));
        });
    }
    __syncthreads();
    auto mw = [&](float v) { return v > -INFINITY && ordered(v) >= cut ? whole_weight(v, d.m, T) : 0; };
    draw_row(sr, V, s, row, gmass[tid], d.m, T, red, found, runs, mw, ids + row, prob);
}

// cuts: the call has top-k, top-p or min-p.
static size_t sample_layout(int rows, int V, bool cuts, uint8_t* at, SampleWs& w) {
    const int chunks = (V + LG_CH - 1) / LG_CH;
    w = SampleWs{};
    size_t n = 0;
    auto take = [&](size_t bytes) {
        uint8_t* p = at ? at + n : nullptr;
        n += (bytes + 255) & ~(size_t)255;
        return p;
    };
    const size_t rc = (size_t)rows * chunks;
    w.chunks = chunks;
    w.best = (u64*)take(rc * 8);
    w.mass = (u64*)take(rc * 8);
    if (!cuts) return n;
    w.least = (float*)take(rc * 4);
    w.hmass = (u64*)take(rc * SM_BINS * 8);
    w.rmass = (u64*)take((size_t)rows * SM_BINS * 8);
    w.rcount = (uint32_t*)take((size_t)rows * SM_BINS * 4);
    w.info = (SampleInfo*)take((size_t)rows * sizeof(SampleInfo));
    w.cand = (uint2*)take((size_t)rows * SM_CAND * 8);
    w.lds = (V + 3) & ~3;
    w.s = (float*)take((size_t)rows * w.lds * 4);
    return n;
}

static bool has_cuts(const SamplingDev& s) { return s.temp && (s.top_k || s.top_p || s.min_p); }

size_t sample_workspace(int rows, int V, bool cuts) {
    SampleWs w;
    return sample_layout(rows, V, cuts, nullptr, w);
}

hipError_t launch_sample(hipStream_t st, const float* x, int64_t ldx, int rows, int V, const SamplingDev& s,
                         int32_t* ids, float* probs, uint8_t* ws) {
    SampleWs w;
    const bool cuts = has_cuts(s);
    sample_layout(rows, V, cuts, ws, w);
    const dim3 chunks(w.chunks, rows);
    return with_forms(vec_rows(x, ldx), has_lists(s), [&](auto vec, auto lists) {
        constexpr bool VEC = vec.value, LISTS = lists.value;
        hipError_t e = op_launch(cuts ? k_sample_scale<VEC, LISTS> : k_sample_weights<VEC, LISTS>, chunks, dim3(LG_T), st, x, ldx,
                                 V, s, w);
        if (e != hipSuccess) return e;
        if (!cuts) return op_launch(k_sample_pick<VEC, LISTS>, dim3(rows), dim3(LG_T), st, x, ldx, V, s, w, ids, probs);
        e = op_launch(k_sample_mass, chunks, dim3(LG_T), st, V, s, w, ids, probs);
        if (e != hipSuccess || !(s.top_k || s.top_p)) return e;
        return op_launch(k_sample_cut, chunks, dim3(LG_T), st, V, s, w, ids, probs);
    });
}
