// What the two attention kernels over the paged 8-bit cache share: their
// arguments, a sequence's share of the work and the cut of all work into runs.
//
// Work is a list of tasks (sequence, row tile, key head), in that order, each
// a number of token tiles. The list is cut into equal runs, one per worker (a
// group of warps), whatever the lengths are (they are on the device; every
// warp finds its worker's run by a scan over them). A task that spans workers
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
// 128): from this many on it is the faster one (8 key heads of 128, 32, 48 and 64
// rows, it against kv_rows_kernel: 4 sequences of 16,000 tokens 94, 95 and 101 us
// against 73, 101 and 118 in bf16, 108, 109 and 114 against 83, 117 and 134 in f16;
// 32 of 2000 103, 104 and 106 against 82, 113 and 141, and 121, 122 and 124 against
// 89, 124 and 155; at dim 64 the two meet at 64 rows: 84, 84 and 84 against 56, 76
// and 94 in bf16) unless the whole call is small (kFewTokens). Launches, or says
// how many bytes of workspace it takes.
constexpr int kPromptRows = 48;
// A call is small where its rows make no more tasks of kv_rows_kernel than there
// are SMs, and these have no more than this many tokens together, by the size of
// the block table: 8 heads, 96 rows of one sequence: 20 us against 24 over 2000
// tokens, 53 against 42 over 16,000 (768,000 together).
constexpr int64_t kFewTokens = 1 << 19;
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

// share(b, tiles, tasks): what sequence b adds to the list. A worker gets at
// least `least` tiles (while there are that many). Where workers get many
// tiles, a task's fixed cost counts as `fixed` of them. PIECES: all tasks of a
// sequence have the same number of tiles, and few tasks are cut into pieces.
//
// Every warp does it for itself, a lane for each 32nd of the sequences: two
// memory latencies and a scan by shuffles, no barrier (at a few sequences, where
// it counts, a scan by the whole block took 2.7 us of a 9 us kernel).
template <bool PIECES, class Share>
__device__ Run find_run(int seqs, int worker, int64_t workers, int least, int fixed, const Share& share) {
    const int lane = threadIdx.x & 31;
    const int per = (seqs + 31) >> 5, b0 = lane * per, b1 = min(seqs, b0 + per);
    const auto scan = [&](int64_t x) {  // inclusive
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t u = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += u;
        }
        return x;
    };
    int64_t mine = 0, mine_tasks = 0;
    #pragma unroll 4
    for (int b = b0; b < b1; ++b) {
        int64_t t = 0, k = 0;
        share(b, t, k);
        mine += t, mine_tasks += k;
    }
    int64_t units = scan(mine);
    const int64_t tasks = scan(mine_tasks), tiles = __shfl_sync(0xffffffffu, units, 31);
    Run run = {};
    run.worker = worker;
    run.tasks = __shfl_sync(0xffffffffu, tasks, 31);
    int64_t task0 = tasks - mine_tasks, from = units - mine;
    if (PIECES && 4 * run.tasks <= workers) {
        const int64_t free = workers - run.tasks;  // rounding up costs a task at most one piece
        run.piece = max(static_cast<int64_t>(least), divide(tiles + free - 1, free));
    } else {
        run.fixed = tiles >= 4LL * fixed * workers ? fixed : 0;
    }
    const auto units_of = [&](int64_t t, int64_t k) {
        if (run.piece == 0) return t + run.fixed * k;
        return k > 0 ? k * divide(divide(t, k) + run.piece - 1, run.piece) : 0;
    };
    if (run.piece != 0) {
        mine = 0;
        for (int b = b0; b < b1; ++b) {
            int64_t t = 0, k = 0;
            share(b, t, k);
            mine += units_of(t, k);
        }
        units = scan(mine);
        from = units - mine;
        run.total = __shfl_sync(0xffffffffu, units, 31);
        run.begin = min(static_cast<int64_t>(worker), run.total);
        run.end = min(run.begin + 1, run.total);
    } else {
        from += run.fixed * task0;
        mine += run.fixed * mine_tasks;
        run.total = tiles + run.fixed * run.tasks;
        const int64_t by = max(int64_t{1}, min(workers, divide(tiles, least)));
        run.each = divide(run.total, by);
        run.extra = run.total - run.each * by;
        run.begin = worker < by ? worker * run.each + min(static_cast<int64_t>(worker), run.extra) : run.total;
        run.end = worker < by ? run.begin + run.each + (worker < run.extra) : run.total;
    }
    // The lane whose sequences hold the first unit walks through them.
    int b = b0;
    const bool here = run.begin >= from && run.begin < from + mine;
    if (here) {
        for (; b < b1 - 1; ++b) {
            int64_t t = 0, k = 0;
            share(b, t, k);
            t = units_of(t, k);
            if (run.begin < from + t) break;
            from += t;
            task0 += k;
        }
    }
    const unsigned int who = __ballot_sync(0xffffffffu, here);
    const int src = who ? __ffs(who) - 1 : 0;  // (none: an empty run)
    run.b = __shfl_sync(0xffffffffu, b, src);
    run.from = __shfl_sync(0xffffffffu, from, src);
    run.task0 = __shfl_sync(0xffffffffu, task0, src);
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

// A block scale, or NaN for an infinite one: a score of minus infinity would
// count as a hidden token.
__device__ __forceinline__ float nan_unless_finite(float scale) { return scale + (scale - scale); }

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
