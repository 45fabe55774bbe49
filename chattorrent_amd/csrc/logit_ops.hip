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
__device__ static inline bool allowed(const RowPens& r, int t) {
    return !r.mask || ((r.mask[t >> 5] >> (t & 31)) & 1u);
}

constexpr int ADJ_CH = 4096;
__global__ __launch_bounds__(LG_T) void k_logits_adjust(const float* x, int64_t ldx, int V, SamplingDev s, float* out,
                                                        int64_t ldo) {
    __shared__ int32_t cnt[ADJ_CH], last[ADJ_CH];
    const int row = blockIdx.y, base = blockIdx.x * ADJ_CH;
    const RowPens r = row_pens(s, row);
    const bool lists = gather_lists<ADJ_CH>(s, r, base, cnt, last);
    for (int i = threadIdx.x; i < ADJ_CH; i += LG_T) {
        const int t = base + i;
        if (t >= V) break;
        float v = x[row * ldx + t];
        if (lists) v = adjust_one(v, s, r, cnt[i], last[i]);
        out[row * ldo + t] = allowed(r, t) ? v : -INFINITY;
    }
}

hipError_t launch_logits_adjust(hipStream_t st, const float* x, int64_t ldx, int rows, int V, const SamplingDev& s,
                                float* out, int64_t ldo) {
    hipLaunchKernelGGL(k_logits_adjust, dim3((V + ADJ_CH - 1) / ADJ_CH, rows), dim3(LG_T), 0, st, x, ldx, V, s, out, ldo);
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
constexpr int SM_CH = 4096;
constexpr double SM_ONE = 4398046511104.0;   // 2^42: a row of 2^20 tokens sums to at most 2^62

__device__ static inline float scaled_logit(float a, double inv_temp) {
    if (!(a > -INFINITY)) return -INFINITY;   // NaN too
    if (a == INFINITY) return a;
    const float s = (float)((double)a * inv_temp);
    return fminf(fmaxf(s, -3.4028234663852886e38f), 3.4028234663852886e38f);
}
__device__ static inline double weight(float s, float m) {
    return s == m ? 1.0 : exp((double)s - (double)m);
}
__device__ static inline uint64_t whole_weight(double w) { return (uint64_t)(w * SM_ONE + 0.5); }

// One workgroup a row: the maximum, then the cuts' values 8 bits at a time
// from the top (counts for top-k, weights for top-p, of the values that share
// the bits so far), then the draw, each a pass over the row. A row and its
// lists are read again in every pass.
constexpr int SMR_T = 256;
struct RowScan {
    const float* x;
    const SamplingDev& s;
    RowPens r;
    int V;
    int32_t *cnt, *last;
    // f(token, adjusted) for every token of chunk c, each by one thread, i the token's place in the chunk
    template <class F>
    __device__ void chunk(int c, F&& f) const {
        const int base = c * SM_CH;
        const bool lists = gather_lists<SM_CH>(s, r, base, cnt, last);
        for (int i = threadIdx.x; i < SM_CH; i += LG_T) {
            const int t = base + i;
            float a = -INFINITY;
            if (t < V) {
                a = x[t];
                if (lists) a = adjust_one(a, s, r, cnt[i], last[i]);
                if (!allowed(r, t)) a = -INFINITY;
            }
            f(t, a);
        }
    }
    template <class F>
    __device__ void all(F&& f) const {
        const int n = (V + SM_CH - 1) / SM_CH;
        for (int c = 0; c < n; c++) chunk(c, f);
    }
};

__device__ static inline uint32_t ordered(float v) {
    const uint32_t b = f2u(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ static inline float unordered(uint32_t k) { return u2f((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

__device__ static inline uint64_t wave_sum64(uint64_t v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((unsigned long long)v, o);
    return v;
}
// Sum over the workgroup, to every thread.
__device__ static inline uint64_t block_sum64(uint64_t v, uint64_t* red) {
    v = wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

__global__ __launch_bounds__(LG_T) void k_sample_row(const float* __restrict__ x, int64_t ldx, int V, SamplingDev s,
                                                     int32_t* __restrict__ ids, float* __restrict__ probs) {
    __shared__ int32_t cnt[SM_CH], last[SM_CH];
    __shared__ unsigned long long hist[256], red[4], sel[2];
    __shared__ unsigned long long s_key;
    const int row = blockIdx.x, tid = threadIdx.x;
    const double temp = s.temp ? (double)s.temp[row] : 0.0;
    const bool greedy = !(temp > 0.0);
    const double inv = greedy ? 1.0 : 1.0 / temp;
    const RowScan scan{x + row * ldx, s, row_pens(s, row), V, cnt, last};
    // the maximum, ties to the lower id; 0: nothing above -inf
    if (tid == 0) s_key = 0;
    unsigned long long best = 0;
    scan.all([&](int t, float a) {
        if (a > -INFINITY) {
            const unsigned long long k = ((unsigned long long)ordered(a) << 32) | (0xffffffffu - (uint32_t)t);
            best = k > best ? k : best;
        }
    });
    __syncthreads();
    atomicMax(&s_key, best);
    __syncthreads();
    if (s_key == 0) {
        if (tid == 0) {
            ids[row] = -1;
            if (probs) probs[row] = 0.0f;
        }
        return;
    }
    if (greedy) {
        if (tid == 0) {
            ids[row] = (int32_t)(0xffffffffu - (uint32_t)s_key);
            if (probs) probs[row] = 1.0f;
        }
        return;
    }
    const float m = scaled_logit(unordered((uint32_t)(s_key >> 32)), inv);
    const int k = s.top_k ? s.top_k[row] : 0;
    const double top_p = s.top_p ? (double)s.top_p[row] : 1.0;
    const double min_p = s.min_p ? fmin((double)s.min_p[row], 1.0) : 0.0;   // the maximum itself stays
    uint32_t cut = 0;   // ordered bits of the smallest value kept
    // the cut where the weights (or counts) from the top reach `want`
    auto find = [&](bool by_count, unsigned long long want) {
        uint32_t prefix = 0;
        unsigned long long left = want;
        for (int sh = 24; sh >= 0; sh -= 8) {
            __syncthreads();
            hist[tid] = 0;
            __syncthreads();
            scan.all([&](int t, float a) {
                const float v = scaled_logit(a, inv);
                const uint32_t o = ordered(v);
                if (v > -INFINITY && o >= cut && (sh == 24 || (o >> (sh + 8)) == (prefix >> (sh + 8))))
                    atomicAdd(&hist[(o >> sh) & 255u], by_count ? 1ull : (unsigned long long)whole_weight(weight(v, m)));
            });
            __syncthreads();
            if (tid == 0) {
                int b = 255;
                unsigned long long above = 0;
                while (b > 0 && above + hist[b] < left) above += hist[b--];
                sel[0] = prefix | ((uint32_t)b << sh);
                sel[1] = left - above;
            }
            __syncthreads();
            prefix = (uint32_t)sel[0];
            left = sel[1];
        }
        return prefix;
    };
    auto mass = [&]() {
        uint64_t sum = 0;
        scan.all([&](int t, float a) {
            const float v = scaled_logit(a, inv);
            if (v > -INFINITY && ordered(v) >= cut) sum += whole_weight(weight(v, m));
        });
        return block_sum64(sum, (uint64_t*)red);
    };
    if (k > 0 && k < V) cut = find(true, (unsigned long long)k);
    if (top_p < 1.0) {
        const double want = ceil(top_p * (double)mass());
        cut = find(false, want < 1.0 ? 1ull : (unsigned long long)want);
    }
    auto kept = [&](float a, double& w) {
        const float v = scaled_logit(a, inv);
        if (!(v > -INFINITY) || ordered(v) < cut) return false;
        w = weight(v, m);
        return w >= min_p;
    };
    uint64_t sum = 0;
    scan.all([&](int t, float a) {
        double w;
        if (kept(a, w)) sum += whole_weight(w);
    });
    const uint64_t total = block_sum64(sum, (uint64_t*)red);
    const double u = s.u ? s.u[row] : 0.0;
    const uint64_t target = min((uint64_t)fmax(u * (double)total, 0.0), total - 1);
    // the chunk that holds the target, then the token
    const int n = (V + SM_CH - 1) / SM_CH;
    uint64_t run = 0;
    for (int c = 0; c < n; c++) {
        uint64_t mine = 0;
        scan.chunk(c, [&](int t, float a) {
            double w;
            if (kept(a, w)) mine += whole_weight(w);
        });
        const uint64_t here = block_sum64(mine, (uint64_t*)red);
        if (run + here <= target) {
            run += here;
            continue;
        }
        // tokens in order: 256 at a time
        scan.chunk(c, [&](int t, float a) {
            double w = 0.0;
            const bool in = kept(a, w);
            const uint64_t mw = in ? whole_weight(w) : 0;
            unsigned long long inc = mw;
            for (int o = 1; o < 64; o <<= 1) {
                const unsigned long long y = __shfl_up(inc, o);
                if ((tid & 63) >= o) inc += y;
            }
            __syncthreads();
            if ((tid & 63) == 63) red[tid >> 6] = inc;
            __syncthreads();
            uint64_t before = run + inc - mw;
            for (int q = 0; q < tid >> 6; q++) before += red[q];
            if (before <= target && target < before + mw) {
                ids[row] = t;
                if (probs) probs[row] = (float)(w * SM_ONE / (double)total);
            }
            run += red[0] + red[1] + red[2] + red[3];
        });
        break;
    }
}

size_t sample_workspace(int rows, int V) { return 256; }

hipError_t launch_sample(hipStream_t st, const float* x, int64_t ldx, int rows, int V, const SamplingDev& s,
                         int32_t* ids, float* probs, uint8_t* ws) {
    hipLaunchKernelGGL(k_sample_row, dim3(rows), dim3(LG_T), 0, st, x, ldx, V, s, ids, probs);
    return hipGetLastError();
}
