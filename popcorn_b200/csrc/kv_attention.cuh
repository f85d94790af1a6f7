// What the two attention kernels over the paged 8-bit cache share: their
// arguments, a sequence's share of the work and the cut of all work into runs.
//
// Work is a list of tasks (sequence, row tile, key head), in that order, each
// a number of token tiles. The list is cut into equal runs, one per worker (a
// group of warps), whatever the lengths are (they are on the device; every
// block finds its workers' runs by a scan over them). A task that spans workers
// leaves partial results (maximum, denominator, weighted sum), two slots per
// worker: slot 0 for a task that an earlier worker began, slot 1 for one that a
// later worker ends. They are joined in the workers' order.
#ifndef POPCORN_B200_KV_ATTENTION_CUH
#define POPCORN_B200_KV_ATTENTION_CUH

#include <cmath>

#include "kv.cuh"

namespace pcb {

struct AttnArgs {
    void* out;
    float* lse;
    const void* q;
    int64_t q_tok, q_head;
    const int8_t* k;
    const int8_t* v;
    const float* ks;
    const float* vs;
    const int32_t* table;
    const int32_t* first;
    const int32_t* length;
    int64_t table_pages, pages, window;
    int seqs, tokens, heads, group, dim, page_shift, causal;
    int min_rows, max_rows;  // this kernel's sequences: tokens times group in [min_rows, max_rows]
    float scale_log2;   // scale * log2(e)
    int q_vec;          // query rows start on four-element boundaries
    int by_task;        // join entries are indexed by task (else by worker)
    int entries;
    int4* entry;        // [0]: number of entries; then two words each, per task or worker
    float2* ml;         // [2 workers][rows]: maximum, denominator
    float* part;        // [2 workers][rows][DP]
};

// The kernel for many query rows of one sequence (16-bit types, dim 64 or
// 128): from this many on it is the faster one. Launches, or says how many
// bytes of workspace it takes.
constexpr int kPromptRows = 17;
bool prompt_supported(popcornType_t type, int64_t dim);
cudaError_t run_prompt(popcornType_t type, const AttnArgs& a, void* ws, int64_t* ws_bytes, cudaStream_t stream);
cudaError_t kv_prompt_take_errors(unsigned int* bits);

#ifdef __CUDACC__
constexpr float kLift = 6.0f;   // probabilities are scaled by 2^6
constexpr float kSlack = 8.0f;  // and may exceed the running maximum by 2^8

struct Seq {
    int row0, rows;  // first query token, number of them (0: another kernel's)
    int len;         // tokens
};

__device__ __forceinline__ Seq sequence(const AttnArgs& a, int b, unsigned int* err) {
    Seq s;
    s.row0 = a.first ? a.first[b] : b;
    s.rows = a.first ? a.first[b + 1] - s.row0 : 1;
    if (s.row0 < 0 || s.rows < 0 || s.rows > a.tokens - s.row0) s.rows = 0;
    if (s.rows * a.group < a.min_rows || s.rows * a.group > a.max_rows) s.rows = 0;
    const int64_t most = a.table_pages << a.page_shift;
    int64_t len = a.length[b];
    if (len > most) {
        atomicOr(err, kKvErrAttention);
        len = most;
    }
    s.len = static_cast<int>(max(len, int64_t{0}));
    return s;
}

// Tokens that queries from..to (of the sequence's) may see: the first one,
// rounded down to 16 (inside its page), and the end.
struct Span {
    int lo, hi;
};
__device__ __forceinline__ Span span_of(const AttnArgs& a, const Seq& s, int from, int to) {
    const int64_t pos = static_cast<int64_t>(s.len) - s.rows;  // of query 0
    int64_t hi = a.causal ? min(pos + to + 1, static_cast<int64_t>(s.len)) : s.len;
    hi = max(hi, int64_t{0});
    int64_t lo = a.window > 0 ? max(pos + from + 1 - a.window, int64_t{0}) : 0;
    lo = min(lo, hi);
    return {static_cast<int>(lo) & ~15, static_cast<int>(hi)};
}

// A worker's run of units and where it begins. A worker is a group of warps;
// `workers` of them share the list, worker g gridDim.x + blockIdx.x being group
// g of a block.
//
// Whole runs (many tasks): units are tiles plus `fixed` for each task; every
// worker gets the same number of them, across tasks. Pieces (few tasks): a task
// is cut into `pieces` equal parts and a worker gets one of them (a unit is a
// piece): no worker pays for the beginning and end of two tasks.
struct Run {
    int64_t begin, end, total;
    int64_t each, extra;  // workers get `each` units, the first `extra` of them one more
    int64_t piece;        // tiles of a piece at most (0: whole runs)
    int fixed;
    int worker;
    int b;                // sequence of unit `begin`
    int64_t from, task0;  // first unit and first task of that sequence
    int64_t tasks;        // of all sequences
};

// 64-bit division that takes the 32-bit instruction sequence where it can.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// Where a sequence's tasks begin in the scan over sequences: tiles or pieces
// before it, tasks before it.
template <int THREADS, class Add, class See>
__device__ __forceinline__ void scan_sequences(int seqs, int64_t (&units)[THREADS / 32], int64_t (&tasks)[THREADS / 32],
                                               int64_t& all_units, int64_t& all_tasks, const Add& add, const See& see) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    all_units = all_tasks = 0;
    for (int base = 0; base < seqs; base += THREADS) {
        int64_t mine = 0, mine_tasks = 0;
        if (base + tid < seqs) add(base + tid, mine, mine_tasks);
        int64_t x = mine, y = mine_tasks;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t u = __shfl_up_sync(0xffffffffu, x, o), w = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) x += u, y += w;
        }
        __syncthreads();  // the sums before have been read
        if (lane == 31) units[warp] = x, tasks[warp] = y;
        __syncthreads();
        int64_t before = all_units, before_tasks = all_tasks;
        #pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) before += units[w], before_tasks += tasks[w];
            all_units += units[w], all_tasks += tasks[w];
        }
        see(base + tid, base + THREADS >= seqs, before + x - mine, mine, before_tasks + y - mine_tasks, mine_tasks);
    }
}

// share(b, tiles, tasks): what sequence b adds to the list. A worker gets at
// least `least` tiles (while there are that many). Where workers get many
// tiles, a task's fixed cost counts as `fixed` of them. PIECES: all tasks of a
// sequence have the same number of tiles, and few tasks are cut into pieces.
template <int THREADS, int GROUPS, bool PIECES, class Share>
__device__ Run find_run(int seqs, int least, int fixed, const Share& share) {
    __shared__ int64_t s_units[THREADS / 32], s_tasks[THREADS / 32], s_from[GROUPS], s_task0[GROUPS];
    __shared__ int s_b[GROUPS];
    const int group = threadIdx.x / (THREADS / GROUPS);
    const int64_t workers = static_cast<int64_t>(GROUPS) * gridDim.x;
    Run run = {};
    int64_t begins[GROUPS];
    const auto cut = [&](int64_t units, int64_t by) {
        run.total = units;
        run.each = divide(units, by);
        run.extra = units - run.each * by;
        #pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            const int64_t me = static_cast<int64_t>(g) * gridDim.x + blockIdx.x;
            const bool on = me < by;
            begins[g] = on ? me * run.each + min(me, run.extra) : units;
            if (g == group) {
                run.worker = static_cast<int>(me);
                run.begin = begins[g];
                run.end = on ? run.begin + run.each + (me < run.extra) : units;
            }
        }
    };
    const auto plan = [&](int64_t tiles, int64_t tasks) {
        run.tasks = tasks;
        if (PIECES && 4 * tasks <= workers) {
            const int64_t free = workers - tasks;  // rounding up costs a task at most one piece
            run.piece = max(static_cast<int64_t>(least), divide(tiles + free - 1, free));
            return;
        }
        run.fixed = tiles >= 4LL * fixed * workers ? fixed : 0;
        cut(tiles + run.fixed * tasks, max(int64_t{1}, min(workers, divide(tiles, least))));
    };
    const auto found = [&](int b, int64_t from, int64_t units, int64_t task0) {
        #pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            if (begins[g] >= from && begins[g] < from + units) s_b[g] = b, s_from[g] = from, s_task0[g] = task0;
        }
    };
    int64_t tiles, tasks;
    scan_sequences<THREADS>(seqs, s_units, s_tasks, tiles, tasks, share,
                            [&](int b, bool last, int64_t from, int64_t mine, int64_t task0, int64_t mine_tasks) {
                                // One chunk holds every sequence: this scan is all it takes.
                                if (seqs > THREADS) return;
                                int64_t all = 0, all_tasks = 0;
                                for (int w = 0; w < THREADS / 32; ++w) all += s_units[w], all_tasks += s_tasks[w];
                                plan(all, all_tasks);
                                if (run.piece == 0) found(b, from + run.fixed * task0, mine + run.fixed * mine_tasks, task0);
                            });
    if (seqs > THREADS) plan(tiles, tasks);
    if (run.piece != 0) {
        // Pieces: their number in all, then (or at once) whose this worker's is.
        const auto pieces = [&](int b, int64_t& units, int64_t& mine_tasks) {
            int64_t t = 0;
            share(b, t, mine_tasks);
            units = mine_tasks > 0 ? mine_tasks * divide(divide(t, mine_tasks) + run.piece - 1, run.piece) : 0;
        };
        #pragma unroll
        for (int g = 0; g < GROUPS; ++g) begins[g] = static_cast<int64_t>(g) * gridDim.x + blockIdx.x;
        run.worker = static_cast<int>(static_cast<int64_t>(group) * gridDim.x + blockIdx.x);
        int64_t count = 0;
        scan_sequences<THREADS>(seqs, s_units, s_tasks, count, tasks, pieces,
                                [&](int b, bool last, int64_t from, int64_t mine, int64_t task0, int64_t mine_tasks) {
                                    found(b, from, mine, task0);
                                });
        run.total = count;
        run.begin = min(static_cast<int64_t>(run.worker), count);
        run.end = min(run.begin + 1, count);
    } else if (seqs > THREADS) {
        scan_sequences<THREADS>(seqs, s_units, s_tasks, tiles, tasks, share,
                                [&](int b, bool last, int64_t from, int64_t mine, int64_t task0, int64_t mine_tasks) {
                                    found(b, from + run.fixed * task0, mine + run.fixed * mine_tasks, task0);
                                });
    }
    __syncthreads();
    run.b = s_b[group], run.from = s_from[group], run.task0 = s_task0[group];
    return run;
}

// The worker that owns unit end - 1 (whole runs).
__device__ __forceinline__ int owner_of_last(const Run& run, int64_t end) {
    const int64_t u = end - 1, longer = run.extra * (run.each + 1);
    return static_cast<int>(u < longer ? divide(u, run.each + 1) : run.extra + divide(u - longer, run.each));
}

// Header of the join entries; workers without a split task say so. By the
// first thread of a worker.
__device__ __forceinline__ void clear_entries(const AttnArgs& a, const Run& run) {
    if (run.worker == 0) a.entry[0] = make_int4(static_cast<int>(a.by_task ? run.tasks : a.entries), 0, 0, 0);
    if (!a.by_task) a.entry[1 + 2 * run.worker] = make_int4(0, 0, 0, 0);
}

// Entry of a task that begins with this worker and ends `more` workers later.
// (A `first` that does not ascend can make more tasks than there are entries.)
__device__ __forceinline__ void put_entry(const AttnArgs& a, const Run& run, int64_t task_number, int more, const Seq& s,
                                          int task) {
    const int64_t e = a.by_task ? task_number : run.worker;
    if (e < a.entries) {
        a.entry[1 + 2 * e] = make_int4(more, run.worker, s.row0, s.rows);
        a.entry[2 + 2 * e] = make_int4(task, 0, 0, 0);
    }
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Scales a partial result with maximum m to the joint maximum.
__device__ __forceinline__ float join_factor(float m, float top) { return m == -INFINITY ? 0.0f : exp2_fast(m - top); }

// 1 / denominator; 0 where the row sees nothing (a NaN stays NaN).
__device__ __forceinline__ float inverse(float l) { return l != 0.0f ? 1.0f / l : 0.0f; }

__device__ __forceinline__ void store_lse(const AttnArgs& a, int64_t t, int head, float l, float top) {
    if (a.lse) {
        a.lse[t * (a.heads * a.group) + head] =
            l != 0.0f ? (top - kLift + log2f(l)) * 0.69314718055994531f : -INFINITY;
    }
}

template <typename T>
__device__ __forceinline__ void store_row(const AttnArgs& a, int64_t t, int head, int d, const float (&o)[4], float l,
                                          float top, bool lead) {
    T* out = static_cast<T*>(a.out) + (t * (a.heads * a.group) + head) * a.dim;
    const float inv = inverse(l);
    if (d < a.dim) {
        const float r[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
        store4(out + d, true, r);
    }
    if (lead) store_lse(a, t, head, l, top);
}
#endif

}  // namespace pcb

#endif  // POPCORN_B200_KV_ATTENTION_CUH
