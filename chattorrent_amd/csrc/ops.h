// Launchers of the operators on the caller's own device buffers
// (cache_ops.hip: paged cache; logit_ops.hip: logits and sampling). Shapes are
// validated by the caller (api.hip) before a launch; each launcher returns its
// launch's error.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <tuple>
#include <type_traits>

// Launches `k` and returns this launch's own error. (hipGetLastError would
// also tell of one that an earlier call of the caller's left behind, for work
// that has been queued well.)
template <class... P, class... A>
hipError_t op_launch(void (*k)(P...), dim3 grid, dim3 block, hipStream_t st, A&&... a) {
    std::tuple<std::decay_t<P>...> args(static_cast<A&&>(a)...);
    const hipError_t e = std::apply(
        [&](auto&... x) {
            void* at[] = {(void*)&x...};
            return hipLaunchKernel((const void*)k, grid, block, at, 0, st);
        },
        args);
    if (e != hipSuccess) (void)hipGetLastError();   // told by the return value
    return e;
}

// ------------------------------------------------------------ paged cache ---
// A paged int8 cache (cc_cache): blk bytes per (page, kv head) block, bblk
// bytes of key bounds per page (all kv heads).
struct CacheDev {
    uint8_t* k = nullptr;
    uint8_t* v = nullptr;
    uint8_t* bounds = nullptr;
    const uint32_t* page_table = nullptr;
    const float* rope = nullptr;
    int nKV = 0, D = 0, ng = 0, rot = 0, n_pages = 0, max_pages = 0, blk = 0, bblk = 0, rope_rows = 0;
};

// A launch's jobs, by value in its kernel arguments (no table to upload, and a
// captured launch keeps them): `first` is the job's first unit of work and
// row0 its first row of the call.
constexpr int OP_JOBS = 128;
struct OpJob {
    int32_t slot, past, n, row0, first;
};
struct OpJobs {
    int n = 0, rows = 0, units = 0;
    OpJob j[OP_JOBS];
};

// cc_positions: positions [rows][n] on n axes (null: a row's index in the
// cache), and the axis of pair j, two bits each.
struct AxesDev {
    const int32_t* pos = nullptr;
    int32_t n = 1;
    uint32_t of[8] = {};
};
// cc_marks: of each (page, kv head) block's 64 rows.
struct MarksDev {
    float* weight = nullptr;
    int32_t* token = nullptr;
};
// What cc_kv_append_at adds; first: the number of each job's first token.
struct AppendAt {
    AxesDev axes;
    MarksDev marks;
    int32_t first[OP_JOBS];
};

// units: pages that the jobs' rows touch.
hipError_t launch_kv_append(hipStream_t st, const CacheDev& c, const OpJobs& jobs, const float* k, int64_t ldk,
                            const float* v, int64_t ldv);
hipError_t launch_kv_append_at(hipStream_t st, const CacheDev& c, const OpJobs& jobs, const AppendAt& at, const float* k,
                               int64_t ldk, const float* v, int64_t ldv);
// units: pages that lie in the jobs' rows as a whole.
hipError_t launch_kv_bounds(hipStream_t st, const CacheDev& c, const OpJobs& jobs);

// How cc_attend_pages lays a call out: work of a row and kv head is `splits`
// workgroups for each 16 query heads (`tiles`), `per` kept pages each.
constexpr int ATTEND_WAVES = 4, ATTEND_PER = 64 * ATTEND_WAVES;   // one page index a lane
constexpr int ATTEND_SPLITS = 128;   // 32768 pages in workgroups of ATTEND_PER
struct AttendPlan {
    int group = 0, tiles = 0, splits = 0, per = 0;
    int max_seen = 0;             // the most pages that a row sees
    int budget = 0, sink = 0, recent = 0;
    bool scored = false;          // a row sees more pages than it keeps
    int score_blocks = 1;         // workgroups that score a row and kv head's pages
    bool vec = false;             // 16-byte loads of the query and the rope table
    size_t scores = 0, partials = 0, counters = 0, bytes = 0;   // offsets into the workspace, and its size
};
// units: rows.
hipError_t launch_attend_pages(hipStream_t st, const CacheDev& c, const OpJobs& jobs, const AttendPlan& p,
                               const float* q, int64_t ldq, float* out, int64_t ldo, uint8_t* ws);

// How cc_attend_weigh lays a launch out. A job's columns are its (row, query
// head of a kv head) pairs, row by row. A unit of attention is a tile of 16 *
// subs columns of a (job, kv head) over `per` pages; its parts lie in the
// workspace as [unit][sub] pieces of 16 columns.
constexpr int WEIGH_JOBS = 64;
struct WeighJob {
    int32_t slot, past, n, row0;
    int32_t count0;   // the first row that counts
    int32_t fresh;    // the first of the slot's rows whose weights fade in this launch
    int32_t unit0, join0, page0;   // its first attention unit, output join and (kv head, page)
};
struct WeighJobs {
    int n = 0, units = 0, joins = 0, pages = 0;
    WeighJob j[WEIGH_JOBS];
};
struct WeighPlan {
    int group = 0, per = 1, subs = 1, score_cols = 0;
    int chunks = 1;   // of the columns whose weights k_weigh_sums adds up
    bool vec = false, weigh = false;
    float fade = 1.0f;
    size_t ml = 0, parts = 0, scores = 0, q = 0, qs = 0, exps = 0, tot = 0, lines = 0, bytes = 0;   // offsets into the workspace, its size
};
constexpr int FINISH_PAGES = 8;   // pages of a workgroup that adds up weights; a (job, kv head)'s are counted in whole ones
constexpr int WEIGH_JOIN = 256;   // floats of a unit's output that a workgroup joins
// By a job's columns: at most 16; up to 64 (a launch's jobs take as many
// 16-column pieces as the largest of them); more, for eight waves of
// weigh_wave_subs(D) pieces each.
enum WeighKind { WEIGH_FEW, WEIGH_NARROW, WEIGH_WIDE };
inline int weigh_wave_subs(int D) { return D > 128 ? 1 : 2; }
hipError_t launch_weigh(hipStream_t st, const CacheDev& c, const WeighJobs& jobs, const WeighPlan& p, WeighKind kind,
                        const AxesDev& axes, const MarksDev& marks, const float* q, int64_t ldq, float* out, int64_t ldo,
                        uint8_t* ws);

// cc_keep; its lists of moves (evict_words each) lie in the workspace from word
// moves0 on, one for each kv head, where it may have more than EVICT_HERE.
struct EvictJob {
    int32_t slot, rows, keep, seen, room;
    int64_t moves0;
};
constexpr int EVICT_JOBS = 96;
struct EvictJobs {
    int n = 0, room = 0, keep = 0;   // room, keep: the largest of the jobs with lists
    EvictJob j[EVICT_JOBS];
};
constexpr int EVICT_HERE = 64;   // moves that the workgroup which selects makes itself
size_t evict_list_words(const EvictJob& j);
hipError_t launch_evict(hipStream_t st, const CacheDev& c, const EvictJobs& jobs, int max_rows, const MarksDev& marks,
                        int sink, int recent, uint8_t* ws);

// -------------------------------------------------------- logits, sampling ---
// cc_sampling with its pointers typed; null: that part is off.
struct SamplingDev {
    const float *temp, *top_p, *min_p, *rep, *freq, *pres, *bias;
    const int32_t *top_k, *pen_at, *pen_ids, *pen_counts, *bias_at, *bias_ids, *mask_of;
    const uint32_t* mask;
    const double* u;
    float freq_cap;
    int n_pen, n_bias, n_masks, mask_words;
};
hipError_t launch_logits_adjust(hipStream_t st, const float* x, int64_t ldx, int rows, int V, const SamplingDev& s,
                                float* out, int64_t ldo);
// cuts: the call has a temperature with top-k, top-p or min-p.
size_t sample_workspace(int rows, int V, bool cuts);
hipError_t launch_sample(hipStream_t st, const float* x, int64_t ldx, int rows, int V, const SamplingDev& s,
                         int32_t* ids, float* probs, uint8_t* ws);
