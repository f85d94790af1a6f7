// What the two attention kernels over the paged 8-bit cache share: their
// arguments, a sequence's share of the work and the cut of all work into one
// run per block.
//
// Work is a list of tasks (sequence, row tile, key head), in that order, each
// a number of units: its token tiles plus a fixed cost. The list is cut into
// equal runs, one per block, whatever the lengths are (they are on the device;
// every block finds its run by a scan over them). A task that spans blocks
// leaves partial results (maximum, denominator, weighted sum), two slots per
// block: slot 0 for a task that began in an earlier block, slot 1 for one that
// ends in a later block. They are joined in block order.
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
    int by_task;        // join entries are indexed by task (else by block)
    int entries;
    int4* entry;        // [0]: number of entries; then two words each, per task or block
    float2* ml;         // [2 blocks][rows]: maximum, denominator
    float* part;        // [2 blocks][rows][DP]
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

// A block's run of units and where it begins.
struct Run {
    int64_t begin, end, total, blocks;
    int b;                // sequence of unit `begin`
    int64_t from, task0;  // first unit and first task of that sequence
    int64_t tasks;        // of all sequences
};

// share(b, units, tasks): what sequence b adds to the list. A block gets at
// least `least` units (while there are that many).
template <int THREADS, class Share>
__device__ Run find_run(int seqs, int least, const Share& share) {
    constexpr int WARPS = THREADS / 32;
    __shared__ int64_t s_units[WARPS], s_tasks[WARPS], s_from, s_task0;
    __shared__ int s_b;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Run run = {0, 0, 0, 1, 0, 0, 0, 0};
    for (int pass = 0; pass < 2; ++pass) {
        int64_t seen = 0, tasks = 0;
        for (int base = 0; base < seqs; base += THREADS) {
            int64_t mine = 0, mine_tasks = 0;
            if (base + tid < seqs) share(base + tid, mine, mine_tasks);
            int64_t x = mine, y = mine_tasks;
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t u = __shfl_up_sync(0xffffffffu, x, o), w = __shfl_up_sync(0xffffffffu, y, o);
                if (lane >= o) x += u, y += w;
            }
            __syncthreads();
            if (lane == 31) s_units[warp] = x, s_tasks[warp] = y;
            __syncthreads();
            int64_t before = seen, before_tasks = tasks;
            #pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                if (w < warp) before += s_units[w], before_tasks += s_tasks[w];
                seen += s_units[w], tasks += s_tasks[w];
            }
            // One chunk holds every sequence: its scan serves both passes.
            if (seqs <= THREADS || pass == 1) {
                if (seqs <= THREADS) {
                    run.total = seen;
                    run.blocks = max(int64_t{1}, min(static_cast<int64_t>(gridDim.x), seen / least));
                    run.begin = min(static_cast<int64_t>(blockIdx.x), run.blocks) * seen / run.blocks;
                }
                const int64_t from = before + x - mine;
                if (run.begin >= from && run.begin < from + mine) {
                    s_b = base + tid;
                    s_from = from;
                    s_task0 = before_tasks + y - mine_tasks;
                }
            }
        }
        run.total = seen;
        run.tasks = tasks;
        run.blocks = max(int64_t{1}, min(static_cast<int64_t>(gridDim.x), seen / least));
        const int64_t me = min(static_cast<int64_t>(blockIdx.x), run.blocks);
        run.begin = me * seen / run.blocks;
        run.end = min(me + 1, run.blocks) * seen / run.blocks;
        if (seqs <= THREADS) break;
    }
    __syncthreads();
    run.b = s_b, run.from = s_from, run.task0 = s_task0;
    return run;
}

// The block that owns the last of units [.., end): block c owns units
// [c total / blocks, (c + 1) total / blocks).
__device__ __forceinline__ int owner_of_last(const Run& run, int64_t end) {
    return static_cast<int>((end * run.blocks - 1) / run.total);
}

// Header of the join entries; blocks without a split task say so.
__device__ __forceinline__ void clear_entries(const AttnArgs& a, const Run& run) {
    if (blockIdx.x == 0) a.entry[0] = make_int4(static_cast<int>(a.by_task ? run.tasks : gridDim.x), 0, 0, 0);
    if (!a.by_task) a.entry[1 + 2 * blockIdx.x] = make_int4(0, 0, 0, 0);
}

// Entry of a task that begins in this block and ends `more` blocks later.
// (A `first` that does not ascend can make more tasks than there are entries.)
__device__ __forceinline__ void put_entry(const AttnArgs& a, int64_t task_number, int more, const Seq& s, int task) {
    const int64_t e = a.by_task ? task_number : blockIdx.x;
    if (e < a.entries) {
        a.entry[1 + 2 * e] = make_int4(more, blockIdx.x, s.row0, s.rows);
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
