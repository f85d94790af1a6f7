// Attention over the paged 8-bit cache for many query rows of one sequence
// (prompt chunks), f16 and bf16, dim 64 or 128: tcgen05 on f16 operands.
//
// Rows are a sequence's queries times the heads that share a key head. A task
// is 256 of them, two tiles of 128 (the tensor instruction's M), against all
// tokens they see in tiles of 128; what it has to do is 4 dim flops a
// (row, token) pair, so it is bound by the tensor cores and, almost as
// closely, by one exponential a pair (16 a cycle and SM: 2048 cycles for the
// 256 x 128 pairs of a step, the same as its two products take).
//
//   scores S = Q K^T: Q as f16 in shared memory (each row scaled by a power
//       of two, exact for f16, and for bf16 down to 2^-24 of the row's largest
//       element), key codes as f16 (exact), f32 sums in tensor memory
//   P = exp2(S ks f + log2(vs) - m): the block scales are constant over 16
//       tokens at least; written over S in tensor memory, for bf16 as one f16 (an
//       eighth of the outputs' own rounding), for f16 as two, the leading 11 bits
//       and the rest, each with a product of its own
//   O += P V: value codes as f16 (exact), transposed on the way into shared
//       memory, f32 sums in tensor memory
//
// Warps 0-3 and 4-7 are the softmax of the two tiles (a thread owns a row, so
// maxima and sums need no exchange), 8-14 convert codes, and one thread of warp
// 15 issues the products: while one tile's softmax runs, the tensor cores work
// on the other's. (Issued by the softmax's own threads the products held them
// up, 2000 cycles a step: the queue is short.) Codes come into shared memory by
// asynchronous copies, so that all loops here are short ones: 16 warps in four
// roles live on one instruction cache, and with the conversion unrolled over
// registers they waited for it more than for anything else. The maximum moves
// only when a score exceeds it by 2^8 (then the thread rescales O in tensor
// memory), as in kv_attention.cu, whose scaling conventions, work split and
// partial results these are.
//
// Measured, with the join: two sequences of 1024 new and 4000 cached tokens, 32
// query heads on 8 of 128: bf16 246 us, 616 TFLOP/s, f16 290 us. (With one f16 for
// a probability f16 took 246 us too, but its results were 2.8e-4 off those in 64
// bits, where rounding to f16 alone makes 2.1e-4, as much as kv_rows_kernel gives.)
// For bf16 the conversion sets the pace, 5000 cycles a step, with the softmax close
// behind (3700 and a wait for the scores); for f16 the softmax does. Tried and
// slower in bf16: an eighth converting warp (the softmax's registers spill, 294 us;
// with registers shared out by setmaxnreg 267 us), warps apart for keys and values
// (341 us).
//
// Every wait is bounded (sm100.cuh); one that runs out sets error bit 0x8000
// and ends the block.
#include <type_traits>

#include "kv_attention.cuh"
#include "sm100.cuh"

namespace pcb {
namespace {

using namespace sm100;

__device__ unsigned int g_prompt_err = 0;
constexpr unsigned int kErrWait = 0x8000u;

constexpr int kTile = 128;          // rows of a tile, tokens of a step
constexpr int kRows = 2 * kTile;    // rows of a task
constexpr int kSoftWarps = 8, kConvWarps = 7, kIssue = kSoftWarps + kConvWarps;
constexpr int kConvThreads = 32 * kConvWarps;
constexpr int kPThreads = 32 * (kIssue + 1);
constexpr int kStages = 2;
constexpr int kScaleRing = 4;
constexpr int kFixedUnits = 2;      // a task's fixed cost in steps

// Barriers, 8 bytes each.
enum Bar { kKFull = 0, kKEmpty = 2, kVFull = 4, kVEmpty = 6, kSFull = 8, kPReady = 10, kODone = 12, kQReady = 14, kDrain = 16, kBars = 17 };

template <int DP>
struct Lay {  // shared memory, bytes; operand tiles in 128-byte swizzled rows
    static constexpr int kQTile = DP / 64 * kTile * 128;
    static constexpr int kKStage = DP / 64 * kTile * 128;
    static constexpr int kVStage = 2 * DP * 128;
    static constexpr int kQ = 0;
    static constexpr int kK = kQ + 2 * kQTile;
    static constexpr int kV = kK + kStages * kKStage;
    static constexpr int kRawK = kV + kStages * kVStage;    // codes of a step as they are
    static constexpr int kRawV = kRawK + kTile * DP;
    static constexpr int kScales = kRawV + kTile * DP;      // [ring][8] {ks, log2 vs, 1 / vs}
    static constexpr int kBytes = kScales + kScaleRing * 8 * 16;
    static constexpr int kAlloc = kBytes + 1024;            // the tiles start on 1024 bytes
};

template <typename T>
using Pair = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
// Probabilities as two f16: the leading bits and the rest.
template <typename T>
constexpr bool kSplit = std::is_same_v<T, __half>;

struct GroupScale {
    float ks, lv, iv, pad;
};

__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void store_shared16(uint32_t addr, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                 : "memory");
}

__device__ __forceinline__ uint4 load_shared16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint32_t load_shared4(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}

__device__ __forceinline__ uint32_t as_f16(uint32_t biased) {  // halves 1024 + code + 128
    const __half2 c = __half2{__float2half_rn(1152.0f), __float2half_rn(1152.0f)};
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&biased), c);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Two scores times their factor, plus log2 of the value scale.
__device__ __forceinline__ float2 scaled(uint32_t s0, uint32_t s1, float kf, float lv) {
    return __ffma2_rn(make_float2(__uint_as_float(s0), __uint_as_float(s1)), make_float2(kf, kf), make_float2(lv, lv));
}
// The leading 11 bits of x: exact in f16 (from 2^-14 on), and so is x less them in
// f32.
__device__ __forceinline__ float high_bits(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }
// -inf for tokens j, j + 1 outside [see0, see1).
__device__ __forceinline__ void hide(float2& v, int j, int see0, int see1) {
    if (j < see0 || j >= see1) v.x = -INFINITY;
    if (j + 1 < see0 || j + 1 >= see1) v.y = -INFINITY;
}

// Walks a block's run segment by segment; every role walks the same way.
struct Walk {
    const AttnArgs& a;
    const Run& run;
    int64_t at, from, task0;
    int b, rt;
    Seq s;
    Span see;             // of the row tile
    int each, steps;      // units and steps of a task of this row tile
    int task_in_tile;     // key head
    int u0, u1;           // the segment's steps
    bool complete;
    int more;             // blocks after this one that hold the rest
    int64_t task_number;

    __device__ Walk(const AttnArgs& args, const Run& r)
        : a(args), run(r), at(r.begin), from(r.from), task0(r.task0), b(r.b), rt(0) {
        if (at < run.end) s = sequence(a, b, &g_prompt_err), tile_sizes();
    }
    __device__ int row_tiles() const { return (s.rows * a.group + kRows - 1) / kRows; }
    __device__ void tile_sizes() {
        see = span_of(a, s, rt * kRows / a.group, min(s.rows - 1, (rt * kRows + kRows - 1) / a.group));
        steps = max((see.hi - see.lo + kTile - 1) / kTile, 1);
        each = run.fixed + steps;
    }
    __device__ bool next() {
        while (at < run.end) {
            if (s.rows == 0 || rt >= row_tiles()) {
                ++b;
                rt = 0;
                s = sequence(a, b, &g_prompt_err);
                if (s.rows > 0) tile_sizes();
                continue;
            }
            const int64_t units = static_cast<int64_t>(each) * a.heads;
            if (at >= from + units) {
                from += units;
                task0 += a.heads;
                if (++rt < row_tiles()) tile_sizes();
                continue;
            }
            task_in_tile = static_cast<int>(divide(at - from, each));
            const int c0 = static_cast<int>(at - from - static_cast<int64_t>(task_in_tile) * each);
            const int c1 = static_cast<int>(min(static_cast<int64_t>(each), c0 + (run.end - at)));
            at += c1 - c0;
            u0 = max(0, c0 - run.fixed);
            u1 = c1 - run.fixed;
            if (u1 <= 0) continue;
            complete = u0 == 0 && u1 == steps;
            more = complete ? 0 : owner_of_last(run, from + static_cast<int64_t>(task_in_tile + 1) * each) - run.worker;
            task_number = task0 + task_in_tile;
            return true;
        }
        return false;
    }
    __device__ int tiles() const { return s.rows * a.group - rt * kRows > kTile ? 2 : 1; }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kPThreads, 1) kv_prompt_kernel(const AttnArgs a) {
    using L = Lay<DP>;
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t bars[kBars];
    __shared__ uint32_t s_tmem;
    const uint32_t smem = (smem_addr(raw) + 1023u) & ~1023u;
    GroupScale* const ring = reinterpret_cast<GroupScale*>(raw + (smem - smem_addr(raw)) + L::kScales);
    const uint32_t bar0 = smem_addr(bars);
    const auto bar = [&](int which, int i) { return bar0 + 8u * (which + i); };
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned int* const err = &g_prompt_err;
    // A warp's lanes go on together, or none does.
    const auto wait = [&](int which, int i, int turn) {
        return __all_sync(0xffffffffu, mbar_wait(bar(which, i), turn & 1, err, kErrWait)) != 0;
    };

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(kKFull, i), kConvThreads);
            mbar_init(bar(kKEmpty, i), 1);
            mbar_init(bar(kVFull, i), kConvThreads);
            mbar_init(bar(kVEmpty, i), 1);
            mbar_init(bar(kSFull, i), 1);
            mbar_init(bar(kPReady, i), kTile);
            mbar_init(bar(kODone, i), 1);
            mbar_init(bar(kQReady, i), kTile);
        }
        mbar_init(bar(kDrain, 0), 1);
        fence_barrier_init();
    }
    // Tensor memory is taken only when the kernel before has ended, and the one
    // after may start only when it has been taken: neither can hold columns
    // that the other waits for.
    pdl_wait();
    if (warp == kIssue) {
        tmem_alloc(smem_addr(&s_tmem), 512);
        tmem_relinquish();
    }
    const Run run = find_run<false>(a.seqs, blockIdx.x, gridDim.x, 1, kFixedUnits, [&](int b, int64_t& steps, int64_t& tasks) {
        const Seq s = sequence(a, b, &g_prompt_err);
        for (int r = 0; r < s.rows * a.group; r += kRows) {
            const Span see = span_of(a, s, r / a.group, min(s.rows - 1, (r + kRows - 1) / a.group));
            steps += static_cast<int64_t>(max((see.hi - see.lo + kTile - 1) / kTile, 1)) * a.heads;
            tasks += a.heads;
        }
    });
    if (tid == 0) clear_entries(a, run);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = s_tmem;
    // Columns: S and P of the two tiles at 0 and 128, O at 256 and 384.

    Walk walk(a, run);
    if (warp < kSoftWarps) {
        // ----------------------------------------------------------- softmax
        const int m = warp >> 2;                    // tile
        const int row = tid & (kTile - 1);
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);  // this warp's 32 lanes
        const uint32_t s_col = lanes + 128 * m, o_col = lanes + 256 + 128 * m;
        int steps_done = 0;                         // of this tile, over all segments
        int kt = 0;                                 // steps of the block, both tiles
        bool good = true;
        while (good && walk.next()) {
            const int n = walk.u1 - walk.u0;
            if (m >= walk.tiles()) {
                kt += n;
                continue;
            }
            const int r = walk.rt * kRows + m * kTile + row;
            const int tok = r / a.group, hd = r - tok * a.group;
            const bool valid = r < walk.s.rows * a.group;
            const int head = walk.task_in_tile * a.group + hd;
            // --- the query row: a power of two brings its largest element to [2^9, 2^10)
            float fac;
            {
                // (held whole: one memory latency)
                const T* q = static_cast<const T*>(a.q) + (walk.s.row0 + tok) * a.q_tok + head * a.q_head;
                Pair<T> x[DP / 2];
                #pragma unroll
                for (int d = 0; d < DP / 2; ++d) x[d].x = x[d].y = from_f32<T>(0.0f);
                if (valid && a.q_vec != 0) {
                    #pragma unroll
                    for (int d = 0; d < DP / 2; d += 2) {
                        *reinterpret_cast<uint2*>(&x[d]) = *reinterpret_cast<const uint2*>(q + 2 * d);
                    }
                } else if (valid) {
                    #pragma unroll
                    for (int d = 0; d < DP / 2; ++d) x[d].x = q[2 * d], x[d].y = q[2 * d + 1];
                }
                Pair<T> most = __habs2(x[0]);
                #pragma unroll
                for (int d = 1; d < DP / 2; ++d) most = __hmax2_nan(most, __habs2(x[d]));
                const T largest_q = __hmax_nan(most.x, most.y);
                const float top = to_f32(largest_q);
                const bool bad = !(top <= 3.4028234663852886e38f);
                const int e = max(-126, min(120, 9 + 127 - static_cast<int>(__float_as_uint(top) >> 23)));
                const float up = bad ? 0.0f : __int_as_float((127 + e) << 23);
                const uint32_t base = smem + L::kQ + m * L::kQTile + row * 128;
                #pragma unroll
                for (int d = 0; d < DP; d += 8) {
                    uint32_t w[4];
                    #pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const Pair<T> v = x[d / 2 + j];
                        w[j] = bad ? 0u : pack_f16(to_f32(v.x) * up, to_f32(v.y) * up);
                    }
                    store_shared16(base + (d / 64) * (kTile * 128) + ((((d % 64) / 8) ^ (row & 7)) << 4), w);
                }
                fac = bad ? __int_as_float(0x7fffffff) : __int_as_float((127 - e) << 23) * a.scale_log2;
            }
            fence_async_shared();
            mbar_arrive(bar(kQReady, m));

            const int64_t pos = static_cast<int64_t>(walk.s.len) - walk.s.rows + tok;
            int see1 = a.causal ? static_cast<int>(max(pos + 1, int64_t{0})) : walk.s.len;
            int see0 = a.window > 0 ? static_cast<int>(max(pos + 1 - a.window, int64_t{0})) : 0;
            see1 = min(see1, walk.s.len);
            if (!valid) see0 = 0, see1 = INT32_MAX;  // (never stored: no reason to mask)
            if (see1 <= see0) fac = 0.0f;
            float top = -INFINITY, den = 0.0f;
            for (int i = 0; i < n; ++i, ++steps_done, ++kt) {
                if (!(good = wait(kSFull, m, steps_done))) break;
                tc_fence_after();
                const GroupScale* gs = ring + (kt % kScaleRing) * 8;
                const int j0 = walk.see.lo + (walk.u0 + i) * kTile;
                const bool whole = __all_sync(0xffffffffu, see0 <= j0 && j0 + kTile <= see1);
                // --- maximum; loops over 32 columns stay loops, for the
                // instruction cache's sake, and load one round ahead.
                uint32_t xa[32], xb[32];
                float best = -INFINITY;
                const auto largest = [&](auto masked, const uint32_t (&x)[32], int c) {
                    #pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float kf = gs[2 * c + h].ks * fac, lv = gs[2 * c + h].lv;
                        float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                        #pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            float2 v = scaled(x[16 * h + j], x[16 * h + j + 1], kf, lv);
                            if (decltype(masked)::value) hide(v, j0 + 32 * c + 16 * h + j, see0, see1);
                            most[j / 2 % 4] = fmaxf(most[j / 2 % 4], fmaxf(v.x, v.y));
                        }
                        best = fmaxf(best, fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])));
                    }
                };
                tmem_ld_32x32b_x32(s_col, xa);
                tmem_wait_ld(xa);
                const auto maximum = [&](auto masked) {
                    #pragma unroll 1
                    for (int c = 0; c < 4; c += 2) {
                        tmem_ld_32x32b_x32(s_col + 32 * (c + 1), xb);
                        largest(masked, xa, c);
                        tmem_wait_ld(xb);
                        tmem_ld_32x32b_x32(s_col + 32 * (c ^ 2), xa);  // the last round fetches the first columns again
                        largest(masked, xb, c + 1);
                        tmem_wait_ld(xa);
                    }
                };
                if (whole) maximum(std::false_type{});
                else maximum(std::true_type{});
                const bool grow = best > top + kSlack;
                if (__any_sync(0xffffffffu, grow)) {
                    const float now = fmaxf(top, best);
                    const float by = join_factor(top, now);
                    top = now;
                    den *= by;
                    if (i > 0) {
                        if (!(good = wait(kODone, m, steps_done - 1))) break;
                        tc_fence_after();
                        #pragma unroll 1
                        for (int c = 0; c < DP / 32; ++c) {
                            uint32_t x[32];
                            tmem_ld_32x32b_x32(o_col + 32 * c, x);
                            tmem_wait_ld(x);
                            #pragma unroll
                            for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * by);
                            tmem_st_32x32b_x32(o_col + 32 * c, x);
                        }
                    }
                }
                // --- probabilities, over the scores (xa holds the first columns)
                const float shift = kLift - (top == -INFINITY ? 0.0f : top);
                const auto weigh = [&](auto masked, const uint32_t (&x)[32], int c) {
                    uint32_t w[16];  // split: the high words of 16 tokens, then their rests
                    #pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const GroupScale g = gs[2 * c + h];
                        const float kf = g.ks * fac, lv = g.lv + shift;
                        float2 sum[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
                        #pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            float2 v = scaled(x[16 * h + j], x[16 * h + j + 1], kf, lv);
                            if (decltype(masked)::value) hide(v, j0 + 32 * c + 16 * h + j, see0, see1);
                            const float2 e = make_float2(exp2_fast(v.x), exp2_fast(v.y));
                            sum[j / 2 % 2] = __fadd2_rn(sum[j / 2 % 2], e);
                            if constexpr (kSplit<T>) {
                                const float2 hi = make_float2(high_bits(e.x), high_bits(e.y));
                                const float2 rest = __ffma2_rn(hi, make_float2(-1.0f, -1.0f), e);
                                w[j / 2] = pack_f16(hi.x, hi.y);
                                w[8 + j / 2] = pack_f16(rest.x, rest.y);
                            } else {
                                w[8 * h + j / 2] = pack_f16(e.x, e.y);
                            }
                        }
                        den = fmaf((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y), g.iv, den);
                        if constexpr (kSplit<T>) tmem_st_32x32b_x16(s_col + 32 * c + 16 * h, w);
                    }
                    if constexpr (!kSplit<T>) tmem_st_32x32b_x16(s_col + 16 * c, w);
                };
                const auto probabilities = [&](auto masked) {
                    #pragma unroll 1
                    for (int c = 0; c < 4; c += 2) {
                        tmem_ld_32x32b_x32(s_col + 32 * (c + 1), xb);
                        weigh(masked, xa, c);
                        tmem_wait_ld(xb);
                        if (c == 0) tmem_ld_32x32b_x32(s_col + 64, xa);
                        weigh(masked, xb, c + 1);
                        if (c == 0) tmem_wait_ld(xa);
                    }
                };
                if (whole) probabilities(std::false_type{});
                else probabilities(std::true_type{});
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(bar(kPReady, m));
            }
            if (!good) break;
            // --- the segment's result
            if (!(good = wait(kODone, m, steps_done - 1))) break;
            tc_fence_after();
            const int64_t slot = (2 * static_cast<int64_t>(blockIdx.x) + (walk.u0 > 0 ? 0 : 1)) * kRows + m * kTile + row;
            const float inv = inverse(den);
            T* out = static_cast<T*>(a.out) + ((walk.s.row0 + tok) * static_cast<int64_t>(a.heads * a.group) + head) * DP;
            #pragma unroll 1
            for (int c = 0; c < DP / 32; ++c) {
                uint32_t x[32];
                tmem_ld_32x32b_x32(o_col + 32 * c, x);
                tmem_wait_ld(x);
                if (!valid) continue;
                if (walk.complete) {
                    #pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        uint4 o;
                        T* e = reinterpret_cast<T*>(&o);
                        #pragma unroll
                        for (int k = 0; k < 8; ++k) e[k] = from_f32<T>(__uint_as_float(x[j + k]) * inv);
                        *reinterpret_cast<uint4*>(out + 32 * c + j) = o;
                    }
                } else {
                    #pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        *reinterpret_cast<uint4*>(a.part + slot * DP + 32 * c + j) =
                            make_uint4(x[j], x[j + 1], x[j + 2], x[j + 3]);
                    }
                }
            }
            if (valid && walk.complete) store_lse(a, walk.s.row0 + tok, head, den, top);
            if (valid && !walk.complete) a.ml[slot] = make_float2(top, den);
            if (tid == 0 && walk.u0 == 0 && (a.by_task || !walk.complete)) {
                put_entry(a, run, walk.task_number, walk.more, walk.s, walk.rt * a.heads + walk.task_in_tile);
            }
            tc_fence_before();  // O has been read: the next segment's products may follow
        }
    } else if (warp < kIssue) {
        // ----------------------------------------------------------- convert
        // A step's tokens are eight groups of 16, each inside one page. The first
        // warp's lanes 0-7 look after a group each: its page index is fetched two
        // steps ahead, its codes' offset and its scales one.
        constexpr int CH = DP / 16;  // 16-byte pieces of a row
        constexpr int WV = DP / 4;   // words of a row
        __shared__ int64_t s_offset[2][8];  // step parity; -1: nothing there
        const int ct = tid - 32 * kSoftWarps;
        const bool scout = ct < 8;
        const int page_mask = (1 << a.page_shift) - 1;
        const auto sync_conv = [&] { asm volatile("bar.sync 1, %0;" ::"n"(kConvThreads) : "memory"); };
        struct Step {
            int h, j0, len;
            int64_t table;  // of the sequence
        };
        int left = 0;  // steps left in the segment
        const auto advance = [&](Step& st) -> bool {
            if (left == 0) {
                if (!walk.next()) return false;
                left = walk.u1 - walk.u0;
                st.h = walk.task_in_tile;
                st.table = static_cast<int64_t>(walk.b) * a.table_pages;
                st.len = min(walk.see.hi, walk.s.len);
                st.j0 = walk.see.lo + walk.u0 * kTile;
            } else {
                st.j0 += kTile;
            }
            --left;
            return true;
        };
        int page = -1;
        float ks = 0.0f, vs = 0.0f;
        bool there = false;
        const auto fetch = [&](const Step& st) {
            const int j = st.j0 + 16 * ct;
            return j < st.len ? a.table[st.table + (j >> a.page_shift)] : -1;
        };
        const auto look_up = [&](const Step& st, int parity) {
            const int j = st.j0 + 16 * ct;
            there = page >= 0 && page < a.pages;
            if (!there && j < st.len) atomicOr(err, kKvErrAttention);
            const int64_t block = static_cast<int64_t>(page) * a.heads + st.h;
            s_offset[parity][ct] = there ? ((block << a.page_shift) + (j & page_mask)) * DP : -1;
            if (there) ks = a.ks[block], vs = a.vs[block];
        };
        // A step's keys or values into their place in shared memory.
        const auto copy = [&](const int8_t* from, int raw_at, int parity) {
            #pragma unroll 2
            for (int i = ct; i < kTile * CH; i += kConvThreads) {
                const int group = i / (16 * CH);
                const int64_t off = s_offset[parity][group];
                cp_async16(smem + raw_at + 16 * i, from + (off < 0 ? 0 : off + 16 * (i % (16 * CH))), off < 0 ? 0 : 16);
            }
            cp_async_commit();
        };
        Step cur = {0, 0, 0, 0}, nxt, after;  // this step, the next, the one after it
        int kt = 0;                           // steps of the block
        bool good = true;
        bool have = advance(cur);
        nxt = cur;
        bool have_next = have && advance(nxt);
        if (have) {
            if (scout) {
                page = fetch(cur);
                look_up(cur, 0);
                page = have_next ? fetch(nxt) : -1;
            }
            sync_conv();
            copy(a.k, L::kRawK, 0);
            copy(a.v, L::kRawV, 0);
            cp_async_wait_group<1>();
            sync_conv();
        }
        // (When a wait runs out the warps go on through their joint barriers, only
        // without the work between them.)
        while (have) {
            after = nxt;
            const bool have_after = have_next && advance(after);
            const int stage = kt % kStages, turn = kt / kStages - 1, parity = (kt + 1) & 1;
            if (good && kt >= kStages) good = wait(kKEmpty, stage, turn);
            if (scout) {
                GroupScale g = {0.0f, -INFINITY, 1.0f, 0.0f};
                if (there) {
                    const bool tiny = fabsf(vs) < kKvSmallestScale;  // all-zero codes
                    g.ks = nan_unless_finite(ks);
                    g.lv = tiny ? -80.0f : __log2f(nan_unless_finite(vs));
                    g.iv = tiny ? 1.0f / kKvSmallestScale
                                : fabsf(vs) <= 3.4028234663852886e38f ? __fdividef(1.0f, vs) : 1.0f;
                }
                ring[(kt % kScaleRing) * 8 + ct] = g;
                if (have_next) look_up(nxt, parity);
                page = have_after ? fetch(after) : -1;
            }
            #pragma unroll 2
            for (int i = ct; good && i < kTile * CH; i += kConvThreads) {
                const uint4 x = load_shared16(smem + L::kRawK + 16 * i);
                const uint32_t in[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
                uint32_t lo[4], hi[4];
                #pragma unroll
                for (int j = 0; j < 2; ++j) {
                    lo[2 * j] = as_f16(__byte_perm(in[j], 0x64646464u, 0x4140));
                    lo[2 * j + 1] = as_f16(__byte_perm(in[j], 0x64646464u, 0x4342));
                    hi[2 * j] = as_f16(__byte_perm(in[2 + j], 0x64646464u, 0x4140));
                    hi[2 * j + 1] = as_f16(__byte_perm(in[2 + j], 0x64646464u, 0x4342));
                }
                const int r = i / CH, piece = i % CH;
                const uint32_t base = smem + L::kK + stage * L::kKStage + (piece / 4) * (kTile * 128) + r * 128;
                const uint32_t unit = 2 * (piece % 4);
                store_shared16(base + ((unit ^ (r & 7)) << 4), lo);
                store_shared16(base + (((unit + 1) ^ (r & 7)) << 4), hi);
            }
            fence_async_shared();
            if (good) mbar_arrive(bar(kKFull, stage));
            cp_async_wait_group<0>();
            sync_conv();  // raw keys are free, raw values there
            if (have_next) copy(a.k, L::kRawK, parity);
            if (good && kt >= kStages) good = wait(kVEmpty, stage, turn);
            // V transposed: row d, 64 tokens to a 128-byte row. Lanes take a word's
            // four bytes in different orders, so that eight lanes' stores fall into
            // eight different 16-byte banks.
            #pragma unroll 1
            for (int i = ct; good && i < 16 * WV; i += kConvThreads) {
                const int word = i % WV, oct = i / WV;
                uint32_t q[8];
                #pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = load_shared4(smem + L::kRawV + (8 * oct + j) * DP + 4 * word);
                #pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t byte = (j + (word >> 1)) & 3;
                    const uint32_t sel = byte | (byte + 4) << 8;
                    uint32_t w[4];
                    #pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t x = __byte_perm(q[2 * k], q[2 * k + 1], sel);
                        w[k] = as_f16((x & 0x00ff00ffu) ^ 0x64806480u);
                    }
                    const uint32_t d = 4 * word + byte;
                    store_shared16(smem + L::kV + stage * L::kVStage + (oct >> 3) * (DP * 128) + d * 128 +
                                       (((oct & 7) ^ (d & 7)) << 4),
                                   w);
                }
            }
            fence_async_shared();
            if (good) mbar_arrive(bar(kVFull, stage));
            cp_async_wait_group<0>();
            sync_conv();  // raw values are free, the next raw keys there
            if (have_next) copy(a.v, L::kRawV, parity);
            nxt = after;
            have = have_next;
            have_next = have_after;
            ++kt;
        }
        cp_async_wait_group<0>();
    } else if (lane == 0) {
        // ------------------------------------------------------------- issue
        constexpr uint32_t id_qk = idesc_f16_f32(kTile, kTile), id_pv = idesc_f16_f32(kTile, DP);
        int kt = 0, segs[2] = {0, 0}, done[2] = {0, 0};
        bool good = true;
        const auto arrived = [&](int which, int i, int turn) { return mbar_wait(bar(which, i), turn & 1, err, kErrWait); };
        const auto scores = [&](int m, int stage) {
            #pragma unroll
            for (int j = 0; j < DP / 16; ++j) {
                const uint32_t off = (j / 4) * (kTile * 128);
                mma_f16_ss(tmem + 128 * m, smem_desc_sw128_kmajor(smem + L::kQ + m * L::kQTile + off) + (j % 4) * 2,
                           smem_desc_sw128_kmajor(smem + L::kK + stage * L::kKStage + off) + (j % 4) * 2, id_qk, j > 0);
            }
            mma_commit(bar(kSFull, m));
        };
        while (good && walk.next()) {
            const int n = walk.u1 - walk.u0, tiles = walk.tiles();
            for (int m = 0; m < tiles && good; ++m) good = arrived(kQReady, m, segs[m]++);
            if (!good || !(good = arrived(kKFull, kt % kStages, kt / kStages))) break;
            tc_fence_after();
            for (int m = 0; m < tiles; ++m) scores(m, kt % kStages);
            mma_commit(bar(kKEmpty, kt % kStages));
            for (int i = 0; i < n && good; ++i, ++kt) {
                const int stage = kt % kStages, next = (kt + 1) % kStages;
                for (int m = 0; m < tiles && good; ++m) {
                    if (m == 0 && !(good = arrived(kVFull, stage, kt / kStages))) break;
                    if (!(good = arrived(kPReady, m, done[m]++))) break;
                    tc_fence_after();
                    #pragma unroll
                    for (int j = 0; j < kTile / 16; ++j) {
                        const uint64_t v = smem_desc_sw128_kmajor(smem + L::kV + stage * L::kVStage + (j / 4) * (DP * 128)) + (j % 4) * 2;
                        const uint32_t p = tmem + 128 * m + (kSplit<T> ? 16 : 8) * j;
                        mma_f16_ts(tmem + 256 + 128 * m, p, v, id_pv, i > 0 || j > 0);
                        if constexpr (kSplit<T>) mma_f16_ts(tmem + 256 + 128 * m, p + 8, v, id_pv, 1);
                    }
                    mma_commit(bar(kODone, m));
                    if (m == tiles - 1) mma_commit(bar(kVEmpty, stage));
                    if (i + 1 < n) {
                        // Over P, so the products that read it have to be done.
                        if (!(good = arrived(kODone, m, done[m] - 1))) break;
                        if (m == 0 && !(good = arrived(kKFull, next, (kt + 1) / kStages))) break;
                        tc_fence_after();
                        scores(m, next);
                        if (m == tiles - 1) mma_commit(bar(kKEmpty, next));
                    }
                }
            }
        }
        // Nothing is in flight any more, or a wait ran out: then it is waited for here.
        mma_commit(bar(kDrain, 0));
        mbar_wait(bar(kDrain, 0), 0, err, kErrWait);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kIssue) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the partial results of split tasks, LANES lanes a row: 8 where there are
// entries for all SMs (all their rows at a time, four to a warp; one after the
// other they took 20 us of a 254 us prompt), 32 where there are few. LANES parts
// at a time: first their maxima and denominators, a lane each, then their sums.
template <typename T, int DP, int LANES>
__global__ void __launch_bounds__(256) kv_prompt_join_kernel(const AttnArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int entries = a.entry[0].x;
    const int4 e = a.entry[1 + 2 * blockIdx.x];
    const int task = a.entry[2 + 2 * blockIdx.x].x;
    if (static_cast<int>(blockIdx.x) >= entries || e.x == 0) return;
    constexpr int VEC = DP / LANES < 4 ? DP / LANES : 4, PIECES = DP / LANES / VEC;
    using Piece = std::conditional_t<VEC == 4, float4, float2>;
    const int l = threadIdx.x % LANES;
    const int r = (blockIdx.y * 256 + threadIdx.x) / LANES;
    const int h = task % a.heads, count = e.x + 1;
    const int row = task / a.heads * kRows + r;
    const bool there = row < e.w * a.group;
    const auto slot = [&](int c) { return static_cast<int64_t>(2 * (e.y + c) + (c == 0 ? 1 : 0)) * kRows + r; };
    float top = -INFINITY, den = 0.0f, sum[PIECES][VEC] = {};
    for (int c0 = 0; c0 < count; c0 += LANES) {
        const int n = min(LANES, count - c0);
        const float2 ml = there && l < n ? a.ml[slot(c0 + l)] : make_float2(-INFINITY, 0.0f);
        float now = fmaxf(top, ml.x);
        #pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, o));
        if (c0 > 0) {
            const float by = join_factor(top, now);
            den *= by;
            #pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                #pragma unroll
                for (int j = 0; j < VEC; ++j) sum[i][j] *= by;
            }
        }
        top = now;
        const float f = join_factor(ml.x, top);
        #pragma unroll 4
        for (int c = 0; c < n; ++c) {
            const float fc = __shfl_sync(0xffffffffu, f, c, LANES);
            den = fmaf(__shfl_sync(0xffffffffu, ml.y, c, LANES), fc, den);
            if (!there) continue;
            const float* p = a.part + slot(c0 + c) * DP + VEC * l;
            #pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const Piece x = *reinterpret_cast<const Piece*>(p + LANES * VEC * i);
                #pragma unroll
                for (int j = 0; j < VEC; ++j) sum[i][j] = fmaf(reinterpret_cast<const float*>(&x)[j], fc, sum[i][j]);
            }
        }
    }
    if (!there) return;
    const int tok = row / a.group, head = h * a.group + row - tok * a.group;
    const float inv = inverse(den);
    T* out = static_cast<T*>(a.out) + ((e.z + tok) * static_cast<int64_t>(a.heads * a.group) + head) * DP + VEC * l;
    #pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        alignas(8) T o[VEC];
        #pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = from_f32<T>(sum[i][j] * inv);
        if constexpr (VEC == 4) {
            *reinterpret_cast<uint2*>(out + LANES * VEC * i) = *reinterpret_cast<const uint2*>(o);
        } else {
            *reinterpret_cast<uint32_t*>(out + LANES * VEC * i) = *reinterpret_cast<const uint32_t*>(o);
        }
    }
    if (l == 0) store_lse(a, e.z + tok, head, den, top);
}

template <typename T, int DP>
cudaError_t run_sized(AttnArgs a, void* ws, int64_t* ws_bytes, cudaStream_t stream) {
    using L = Lay<DP>;
    const int64_t grid = device_sm_count();
    const int64_t entry_bytes = (1 + 2 * grid) * sizeof(int4), ml_bytes = 2 * grid * kRows * sizeof(float2);
    if (ws_bytes != nullptr) {
        *ws_bytes = entry_bytes + ml_bytes + 2 * grid * kRows * DP * sizeof(float);
        return cudaSuccess;
    }
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !__atomic_load_n(&ready[dev], __ATOMIC_RELAXED)) {
        e = cudaFuncSetAttribute(kv_prompt_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAlloc);
        if (e != cudaSuccess) return e;
        if (dev < 64) __atomic_store_n(&ready[dev], true, __ATOMIC_RELAXED);
    }
    const int64_t tasks = a.heads * (static_cast<int64_t>(a.tokens) * a.group / kRows + a.seqs);
    a.by_task = tasks <= grid ? 1 : 0;
    a.entries = static_cast<int>(a.by_task ? tasks : grid);
    a.entry = static_cast<int4*>(ws);
    a.ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + entry_bytes);
    a.part = reinterpret_cast<float*>(static_cast<char*>(ws) + entry_bytes + ml_bytes);
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = pdl_config(dim3(static_cast<unsigned>(grid)), dim3(kPThreads), L::kAlloc, stream, attr);
    e = cudaLaunchKernelEx(&cfg, kv_prompt_kernel<T, DP>, a);
    if (e != cudaSuccess) return e;
    const int lanes = 8 * a.entries <= 2 * grid ? 32 : 8;
    cfg.gridDim = dim3(static_cast<unsigned>(a.entries), kRows * lanes / 256);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    return lanes == 8 ? cudaLaunchKernelEx(&cfg, kv_prompt_join_kernel<T, DP, 8>, a)
                      : cudaLaunchKernelEx(&cfg, kv_prompt_join_kernel<T, DP, 32>, a);
}

}  // namespace

bool prompt_supported(popcornType_t type, int64_t dim) {
    return (type == POPCORN_TYPE_F16 || type == POPCORN_TYPE_BF16) && (dim == 64 || dim == 128);
}

cudaError_t run_prompt(popcornType_t type, const AttnArgs& a, void* ws, int64_t* ws_bytes, cudaStream_t stream) {
    if (type == POPCORN_TYPE_F16) {
        return a.dim == 64 ? run_sized<__half, 64>(a, ws, ws_bytes, stream) : run_sized<__half, 128>(a, ws, ws_bytes, stream);
    }
    return a.dim == 64 ? run_sized<__nv_bfloat16, 64>(a, ws, ws_bytes, stream)
                       : run_sized<__nv_bfloat16, 128>(a, ws, ws_bytes, stream);
}

cudaError_t kv_prompt_take_errors(unsigned int* bits) {
    const unsigned int zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(bits, g_prompt_err, sizeof(unsigned int));
    if (e == cudaSuccess && *bits != 0) e = cudaMemcpyToSymbol(g_prompt_err, &zero, sizeof(unsigned int));
    return e;
}

}  // namespace pcb
