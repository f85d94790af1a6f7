// A mixture-of-experts layer for a few tokens on per-channel int8 experts:
//   z = x Wr^T,  p = softmax(z),  the top_k largest p of each token,
//   out[m] = sum over its experts e of p'_e * (silu(x Wg_e^T) * (x Wu_e^T)) Wd_e^T.
// What it cannot do without is one read of the chosen experts' codes, 3 K F
// bytes each; it is bound by HBM. Three launches, overlapped by programmatic
// dependent launch:
//  1. route_kernel: the logits, one block per expert and eight tokens, and the
//     activations as fixed point.
//  2. up_kernel: every block picks the experts itself from the logits (a few
//     KB, cheaper than a launch), then walks over (chosen expert, 32 rows of
//     gate and of up) items and writes silu(g) u as fixed point.
//  3. down_kernel: a block owns up to 32 output channels at a time and goes
//     through all chosen experts, so that a token's sum over its experts needs no
//     other block.
// Measured in a graph: one token, 2 of 16 experts of 4096 x 11008: 56 us, 4.8 TB/s;
// 16 tokens, 6 of 64 experts of 2048 x 1424 each: 99 us, 4.5 TB/s. By themselves,
// with cold caches, the kernels read at 5.0 (up, 37 us) and 4.0 TB/s (down, 23 us)
// and at 4.7 (63 us) and 4.0 TB/s (41 us): their starts, the ends of their blocks
// and, in down, the wait for the first codes are inside.
//
// Products. mma s8 x s8 -> s32 with the codes as they are: 16 weight rows are
// the M side; the eight columns of the N side are two tokens times the four
// balanced base-256 digits of 30-bit fixed point. Sums are exact integers and
// join in double or f32, so the result's error is f32 rounding. Codes come through
// rings of shared memory that each warp fills by asynchronous copies and reads
// alone; digits are read in 16-byte loads from L2. Columns of the product may be
// taken in any order, so lane (g, t) = (lane / 4, lane % 4) takes piece t of each
// 64-column window of both, the words of which feed two 32-deep steps. The
// activations' fixed point has one power of two per token, the hidden values' one
// for each 32 rows that an item covers: columns 64 w + 16 t + 8 s + i (t < 4, i < 8),
// which are the columns of step s of window w in the next product.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "mma_frag.cuh"
#include "popcorn_serve.h"

namespace pcb {
namespace {

constexpr int kDownWarps = 16, kDownThreads = 32 * kDownWarps;
constexpr int kDownShared = 208 * 1024;  // dynamic shared memory beside the routing lists
constexpr int kMoeThreads = 256;
constexpr int kMoeWarps = kMoeThreads / 32;
constexpr int kWindows = 4;       // windows of a stage: 256 columns of 16 rows
constexpr int kColumns = 64 * kWindows;
constexpr int kStageBytes = 16 * kColumns;  // [window][16 rows][64 bytes]
constexpr int kMoeTokens = 64;    // tokens of one pass
constexpr int kMoeExperts = 256;
constexpr int kMoeTop = 16;
constexpr int kMagicBits = 0x4B400000;   // 1.5 2^23 as f32
constexpr float kMagic = 12582912.0f;

struct MoeArgs {
    float* out;
    int* experts;      // [M, top]
    float* weights;    // [M, top]
    const float* x;
    const float* router;
    const int8_t* qg;
    const float* sg;
    const int8_t* qu;
    const float* su;
    const int8_t* qd;
    const float* sd;
    float* logits;     // [M, E]
    int8_t* xd;        // [M][4][kp] digits of x
    float* xs;         // [M] its unit
    int8_t* hd;        // [M top][4][fp] digits of the hidden values
    float* hs;         // [M top][fp / 32] their units (kp, fp: K, F rounded up to whole stages)
    float* h;          // [M top][F] hidden values (plain kernels only)
    int M, K, F, E, top, renorm, kp, fp;
    int rows;          // output channels of a tile of the down product
};

// Fixed point of values up to m in magnitude: 2^s brings m to [2^29, 2^30)
// (as two factors, since s goes up to 149, where the unit 2^-s is f32's
// smallest number). Zero gives digits 0; a non-finite m digits 0 and unit NaN.
struct Fixed {
    float up, more, unit;
};
__device__ __forceinline__ Fixed fixed_for(float m, bool bad) {
    if (bad) return {0.0f, 0.0f, __int_as_float(0x7fffffff)};
    const int s = max(-98, min(149, 29 + 127 - static_cast<int>(__float_as_uint(m) >> 23)));
    const int s0 = min(s, 126);
    return {__int_as_float((127 + s0) << 23), __int_as_float((127 + s - s0) << 23), ldexpf(1.0f, -s)};
}
// The four balanced digits of v, lowest byte first.
__device__ __forceinline__ uint32_t digits_of(float v, const Fixed& f) {
    return (static_cast<uint32_t>(__float2int_rn(v * f.up * f.more)) + 0x80808080u) ^ 0x80808080u;
}
__device__ __forceinline__ bool not_finite(float v) { return !(fabsf(v) <= 3.4028234663852886e38f); }

// ------------------------------------------------------------------ routing
// Block e < E: logits of expert e for tokens 8 y .. 8 y + 7. Blocks behind them
// (y = 0): the digits of one token each. The router is f32 and may be what the
// kernel ahead writes: its rows are read after the wait like everything else, and
// only fetched into L2 before it. (One token through 2 of 16 experts of 4096 x
// 11008, called from Python: 58.1 us, 58.7 without the fetch, 57.5 when the rows
// were read before the wait.)
constexpr int kRouteThreads = 256, kRouteWarps = kRouteThreads / 32;
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const MoeArgs a) {
    constexpr int HELD = 4;  // float4 pieces of the router's row per thread: 4096 columns
    __shared__ float part[kRouteWarps][8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    const int e = blockIdx.x;
    const bool vec =
        a.K % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.router) | reinterpret_cast<uintptr_t>(a.x)) & 15u) == 0;
    const float* w = a.router + static_cast<int64_t>(e) * a.K;
    float4 held[HELD];
    if (e < a.E && tid == 0) prefetch_l2_range(w, sizeof(float) * min(a.K, 4 * HELD * kRouteThreads), 0, 1);
    pdl_wait();
    if (e >= a.E) {
        const int m = e - a.E;
        if (blockIdx.y != 0 || a.xd == nullptr) return;
        const float* x = a.x + static_cast<int64_t>(m) * a.K;
        // Four columns at a time, the first ones held between maximum and digits.
        const auto four = [&](int k) {
            if (k >= a.K) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            return vec ? *reinterpret_cast<const float4*>(x + k) : make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
        };
        float top = 0.0f;
        bool bad = false;
        const auto look = [&](const float4& v) {
            top = fmaxf(fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
            bad = bad || not_finite(v.x) || not_finite(v.y) || not_finite(v.z) || not_finite(v.w);
        };
        #pragma unroll
        for (int i = 0; i < HELD; ++i) held[i] = four(4 * (tid + i * kRouteThreads));
        #pragma unroll
        for (int i = 0; i < HELD; ++i) look(held[i]);
        for (int k = 4 * (tid + HELD * kRouteThreads); k < a.K; k += 4 * kRouteThreads) look(four(k));
        top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
        if (lane == 0) part[warp][0] = top;
        const bool any_bad = __syncthreads_or(bad) != 0;
        #pragma unroll
        for (int i = 0; i < kRouteWarps; ++i) top = fmaxf(top, part[i][0]);
        const Fixed f = fixed_for(top, any_bad);
        int8_t* d = a.xd + static_cast<int64_t>(m) * 4 * a.kp;
        const auto put = [&](int k, const float4& v) {
            if (k >= a.kp) return;
            const uint32_t y[4] = {any_bad ? 0u : digits_of(v.x, f), any_bad ? 0u : digits_of(v.y, f),
                                   any_bad ? 0u : digits_of(v.z, f), any_bad ? 0u : digits_of(v.w, f)};
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t sel = static_cast<uint32_t>(i | ((i + 4) << 4));
                *reinterpret_cast<uint32_t*>(d + static_cast<int64_t>(i) * a.kp + k) =
                    __byte_perm(__byte_perm(y[0], y[1], sel), __byte_perm(y[2], y[3], sel), 0x5410);
            }
        };
        #pragma unroll
        for (int i = 0; i < HELD; ++i) put(4 * (tid + i * kRouteThreads), held[i]);
        for (int k = 4 * (tid + HELD * kRouteThreads); k < a.kp; k += 4 * kRouteThreads) put(k, four(k));
        if (tid == 0) a.xs[m] = f.unit;
        // Units of the padding of this token's hidden values (its digits meet codes
        // that are zeros and may be anything).
        const int used = (a.F + 63) / 64 * 2, all = a.fp / 32;
        for (int i = tid; i < a.top * (all - used); i += kRouteThreads) {
            const int j = i / (all - used);
            a.hs[(static_cast<int64_t>(m) * a.top + j) * all + used + i - j * (all - used)] = 0.0f;
        }
        return;
    }
    const int m0 = blockIdx.y * 8;
    const int n = min(8, a.M - m0);
    const float* x = a.x + static_cast<int64_t>(m0) * a.K;
    float acc[8] = {};
    const auto add = [&](int k, const float4& q) {
        #pragma unroll
        for (int m = 0; m < 8; ++m) {
            if (m < n) {
                const float4 v = *reinterpret_cast<const float4*>(x + static_cast<int64_t>(m) * a.K + k);
                acc[m] = fmaf(q.x, v.x, fmaf(q.y, v.y, fmaf(q.z, v.z, fmaf(q.w, v.w, acc[m]))));
            }
        }
    };
    if (vec) {
        #pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int k = 4 * (tid + i * kRouteThreads);
            held[i] = k < a.K ? *reinterpret_cast<const float4*>(w + k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        #pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int k = 4 * (tid + i * kRouteThreads);
            if (k < a.K) add(k, held[i]);
        }
        for (int k = 4 * (tid + HELD * kRouteThreads); k < a.K; k += 4 * kRouteThreads) {
            add(k, *reinterpret_cast<const float4*>(w + k));
        }
    } else {
        for (int k = tid; k < a.K; k += kRouteThreads) {
            #pragma unroll
            for (int m = 0; m < 8; ++m) {
                if (m < n) acc[m] = fmaf(w[k], x[static_cast<int64_t>(m) * a.K + k], acc[m]);
            }
        }
    }
    #pragma unroll
    for (int m = 0; m < 8; ++m) {
        if (m < n) {
            #pragma unroll
            for (int o = 16; o > 0; o >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], o);
            if (lane == 0) part[warp][m] = acc[m];
        }
    }
    __syncthreads();
    if (tid < n) {
        float z = 0.0f;
        #pragma unroll
        for (int i = 0; i < kRouteWarps; ++i) z += part[i][tid];
        a.logits[static_cast<int64_t>(m0 + tid) * a.E + e] = z;
    }
}

// What a block knows of the routing. A job is up to 2 NP tokens of one
// expert; the list of positions holds the chosen experts' (token, pick) pairs
// expert by expert, tokens ascending.
struct Routing {
    unsigned int tokens[kMoeExperts][2];            // an expert's tokens, as bits
    short base[kMoeExperts];                        // its first position
    short pair[kMoeTokens * kMoeTop];               // position -> token * top + pick
    unsigned char token[kMoeTokens * kMoeTop];      // position -> token
    unsigned int job[kMoeTokens * kMoeTop];         // expert | position << 8 | tokens << 24
    int jobs;
    short pick[kMoeTokens * kMoeTop];               // pair -> expert
    float weight[kMoeTokens * kMoeTop];             // pair -> weight
};
struct Job {
    int expert, pos, count;
};
__device__ __forceinline__ Job job_of(const Routing& r, int j) {
    const unsigned int x = r.job[j];
    return {static_cast<int>(x & 0xffu), static_cast<int>(x >> 8 & 0xffffu), static_cast<int>(x >> 24)};
}

// One warp: token m's experts. Softmax over all logits; the top ones by
// repeated maxima, the lowest index first among equals. NaN logits count as
// -inf. Writes pick and weight.
__device__ void pick_experts(const MoeArgs& a, int m, Routing& r, int lane) {
    constexpr int PER = kMoeExperts / 32;
    float z[PER];
    float top = -INFINITY;
    #pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane + 32 * i;
        z[i] = e < a.E ? a.logits[static_cast<int64_t>(m) * a.E + e] : -INFINITY;
        top = fmaxf(top, z[i]);
    }
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float sum = 0.0f;
    #pragma unroll
    for (int i = 0; i < PER; ++i) sum += lane + 32 * i < a.E ? expf(z[i] - top) : 0.0f;
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    unsigned int taken = 0;  // bit i: z[i] has been picked
    float mine = 0.0f;       // lane j: probability of pick j
    int mine_e = 0;
    float picked = 0.0f;
    for (int j = 0; j < a.top; ++j) {
        float best = -INFINITY;
        int at = kMoeExperts;
        #pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane + 32 * i;
            const bool open = e < a.E && !(taken >> i & 1u);
            if (open && (at == kMoeExperts || z[i] > best)) best = z[i] == z[i] ? z[i] : -INFINITY, at = e;
        }
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ob = __shfl_xor_sync(0xffffffffu, best, o);
            const int oa = __shfl_xor_sync(0xffffffffu, at, o);
            if (ob > best || (ob == best && oa < at)) best = ob, at = oa;
        }
        if ((at & 31) == lane) taken |= 1u << (at >> 5);
        const float p = expf(best - top) / sum;
        picked += p;
        if (lane == j) mine = p, mine_e = at;
    }
    if (lane < a.top) {
        r.pick[m * a.top + lane] = static_cast<short>(mine_e);
        r.weight[m * a.top + lane] = a.renorm ? mine / picked : mine;
    }
}

// The block's lists from the picks in r.pick.
template <int NP, int THREADS>
__device__ void list_jobs(const MoeArgs& a, Routing& r) {
    const int tid = threadIdx.x;
    for (int e = tid; e < a.E; e += THREADS) r.tokens[e][0] = r.tokens[e][1] = 0;
    __syncthreads();
    for (int i = tid; i < a.M * a.top; i += THREADS) {
        const int m = i / a.top;
        atomicOr(&r.tokens[r.pick[i]][m >> 5], 1u << (m & 31));
    }
    __syncthreads();
    if (tid < 32) {
        int jobs = 0, pos = 0;
        for (int e0 = 0; e0 < a.E; e0 += 32) {
            const int e = e0 + tid;
            const int n = e < a.E ? __popc(r.tokens[e][0]) + __popc(r.tokens[e][1]) : 0;
            const int j = (n + 2 * NP - 1) / (2 * NP);
            int sum = n | j << 16;  // both totals stay under 2^11
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, sum, o);
                if (tid >= o) sum += u;
            }
            const int from = pos + (sum & 0xffff) - n, job = jobs + (sum >> 16) - j;
            if (n) r.base[e] = static_cast<short>(from);
            for (int k = 0; k < j; ++k) {
                r.job[job + k] = static_cast<unsigned int>(e) | static_cast<unsigned int>(from + 2 * NP * k) << 8 |
                                 static_cast<unsigned int>(min(2 * NP, n - 2 * NP * k)) << 24;
            }
            sum = __shfl_sync(0xffffffffu, sum, 31);
            pos += sum & 0xffff;
            jobs += sum >> 16;
        }
        if (tid == 0) r.jobs = jobs;
    }
    __syncthreads();
    for (int i = tid; i < a.M * a.top; i += THREADS) {
        const int m = i / a.top, e = r.pick[i];
        const unsigned int below = (1u << (m & 31)) - 1u;
        const int rank = m < 32 ? __popc(r.tokens[e][0] & below) : __popc(r.tokens[e][0]) + __popc(r.tokens[e][1] & below);
        r.pair[r.base[e] + rank] = static_cast<short>(i);
        r.token[r.base[e] + rank] = static_cast<unsigned char>(m);
    }
    __syncthreads();
}

template <int THREADS>
__device__ void route_tokens(const MoeArgs& a, Routing& r) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int m = warp; m < a.M; m += THREADS / 32) pick_experts(a, m, r, lane);
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < a.M * a.top; i += THREADS) {
            a.experts[i] = r.pick[i];
            a.weights[i] = r.weight[i];
        }
    }
}

// ------------------------------------------------------------- gate and up
// An item is a job's 32 rows of both matrices: two tiles of 16 rows each, of
// which rows 0-7 and 8-15 are runs of eight (the columns that share a unit in
// the next product). A block is an SM's whole load, three workers of four warps,
// each with its own items and barrier; a warp has one of the four tiles and
// streams its rows, from one item into the next, through a ring of its own in
// shared memory by asynchronous copies, 256 bytes of each row (4 KB) a stage:
// 144 KB an SM in flight. (Loads into registers with two or three blocks an SM
// kept at most 96 KB in flight; warps that shared
// the rows and had a quarter of the columns each read 64 bytes a row at a time:
// 38 us against 34 for the two experts of 11008 rows.)
//
// With eight tokens to a job the digits are twice the codes, and each of the four
// warps read all of them. There a warp has 16 rows of both matrices and half of
// the columns, 128 bytes of each row a stage, and two warps' sums are added: 25
// tokens that all pick all 8 experts of 2560 x 6448 took 179 us instead of 221.
constexpr int kUpWarps = 4, kUpThreads = 32 * kUpWarps, kUpWorkers = 3;
template <int NP>
struct Up {
    static constexpr int kStages = NP == 4 ? 3 : 4;
    static constexpr bool kPaired = NP == 4;         // a warp has both matrices' rows, half of the columns
    static constexpr int kTiles = kPaired ? 2 : 1;   // of 16 rows, a warp's
    static constexpr int kWide = kPaired ? 2 : 4;    // windows of a stage
    static constexpr int kParities = NP == 1 ? 2 : 1;  // an item's sums may wait while the next is multiplied
    static constexpr int kBytes = kUpWorkers * kUpWarps * kStages * kStageBytes;
};

__device__ __forceinline__ uint4 load_shared16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}

// One stage: this lane's pieces of its rows, one of every eight (of `bytes` 16,
// or 0 for rows that are not there), from column `col` on, zeros past `end`.
template <int GROUPS, int WIDE>
__device__ __forceinline__ void copy_stage(uint32_t dst, const int8_t* const (&rows)[GROUPS], const int (&bytes)[GROUPS],
                                           int col, int t, int end) {
    if (col + 64 * WIDE <= end) {
        #pragma unroll
        for (int k = 0; k < WIDE; ++k) {
            #pragma unroll
            for (int i = 0; i < GROUPS; ++i) cp_async16(dst + 512 * (GROUPS * k + i), rows[i] + col + 64 * k, bytes[i]);
        }
    } else {
        #pragma unroll
        for (int k = 0; k < WIDE; ++k) {
            const bool in = col + 64 * k + 16 * t < end;
            #pragma unroll
            for (int i = 0; i < GROUPS; ++i) {
                cp_async16(dst + 512 * (GROUPS * k + i), rows[i] + (in ? col + 64 * k : 0), in ? bytes[i] : 0);
            }
        }
    }
}

template <int NP>
__global__ void __launch_bounds__(kUpWorkers* kUpThreads, 1) up_kernel(const MoeArgs a) {
    constexpr int STAGES = Up<NP>::kStages, THREADS = kUpWorkers * kUpThreads;
    extern __shared__ __align__(128) uint8_t s_ring[];
    __shared__ Routing r;
    __shared__ __align__(16) int s_sums[kUpWorkers][Up<NP>::kParities][4][16][8 * NP];  // [item parity][gate 0, gate 1, up 0, up 1][row][token, digit]
    const int worker = threadIdx.x / kUpThreads;
    const int tid = threadIdx.x % kUpThreads, lane = tid & 31, warp = tid >> 5;  // of the worker
    const int g = lane >> 2, t = lane & 3;
    const auto sync_worker = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1 + worker), "n"(kUpThreads) : "memory"); };
    auto& sums = s_sums[worker];
    pdl_launch_dependents();
    pdl_wait();
    route_tokens<THREADS>(a, r);
    list_jobs<NP, THREADS>(a, r);

    const int halves = (a.F + 63) / 64 * 2, stages = a.kp / kColumns;
    const int items = r.jobs * halves;
    const int first = worker * gridDim.x + blockIdx.x, stride = kUpWorkers * gridDim.x;
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(s_ring)) +
                          (worker * kUpWarps + warp) * STAGES * kStageBytes + 16 * lane;
    constexpr int TILES = Up<NP>::kTiles, WIDE = Up<NP>::kWide;
    constexpr bool PAIRED = Up<NP>::kPaired;
    const int half = PAIRED ? 64 * WIDE * (warp >> 1) : 0;  // first column of a stage
    const int8_t* const codes = (!PAIRED && (warp & 2) ? a.qu : a.qg) + 16 * t;

    // The copying side: item, stage of it and this lane's rows g and g + 8.
    int c_item = first, c_s = 0, c_slot = 0;
    const int8_t* rows[2 * TILES] = {};
    int bytes[2 * TILES];
    #pragma unroll
    for (int i = 0; i < 2 * TILES; ++i) bytes[i] = 16;
    const auto rows_of = [&](int item) {
        const int h = item % halves;
        const int f = h / 2 * 64 + 32 * (warp & 1) + 8 * (h & 1) + g;
        const int64_t at = static_cast<int64_t>(job_of(r, item / halves).expert) * a.F;
        rows[0] = codes + (at + min(f, a.F - 1)) * a.K;
        rows[1] = codes + (at + min(f + 16, a.F - 1)) * a.K;
        if constexpr (PAIRED) {
            rows[2] = a.qu + 16 * t + (at + min(f, a.F - 1)) * a.K;
            rows[3] = a.qu + 16 * t + (at + min(f + 16, a.F - 1)) * a.K;
        }
    };
    const auto copy_next = [&] {
        if (c_item < items) {
            copy_stage<2 * TILES, WIDE>(ring + c_slot * kStageBytes, rows, bytes, c_s * kColumns + half, t, a.K);
            if (++c_s == stages) {
                c_s = 0;
                c_item += stride;
                if (c_item < items) rows_of(c_item);
            }
        }
        cp_async_commit();
        c_slot = c_slot == STAGES - 1 ? 0 : c_slot + 1;
    };
    if (first < items) rows_of(first);
    #pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) copy_next();

    int parity = 0, slot = 0;
    for (int item = first; item < items; item += stride, parity ^= Up<NP>::kParities - 1) {
        const Job job = job_of(r, item / halves);
        // This lane's column of the B operand: a digit of a token. (Columns of
        // tokens that the job does not have repeat its last one and are not used.)
        const int8_t* xd[NP];
        #pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int m = r.token[job.pos + min(2 * n + (g >> 2), job.count - 1)];
            xd[n] = a.xd + (static_cast<int64_t>(m) * 4 + (g & 3)) * a.kp + 16 * t + half;
        }
        uint4 b[WIDE][NP];
        const auto load_b = [&](int st) {
            #pragma unroll
            for (int k = 0; k < WIDE; ++k) {
                #pragma unroll
                for (int n = 0; n < NP; ++n) b[k][n] = *reinterpret_cast<const uint4*>(xd[n] + kColumns * st + 64 * k);
            }
        };
        if (NP <= 2) load_b(0);
        int acc[TILES][NP][4] = {};
        for (int st = 0; st < stages; ++st) {
            if (NP > 2) load_b(st);  // (held a stage ahead: 185 us against 179 for the example above)
            cp_async_wait_group<STAGES - 2>();
            __syncwarp();
            copy_next();
            const uint32_t at = ring + slot * kStageBytes;
            slot = slot == STAGES - 1 ? 0 : slot + 1;
            #pragma unroll
            for (int k = 0; k < WIDE; ++k) {
                #pragma unroll
                for (int i = 0; i < TILES; ++i) {
                    const uint32_t from = at + 1024 * (TILES * k + i);
                    const uint4 q0 = load_shared16(from), q1 = load_shared16(from + 512);
                    const uint32_t lo[4] = {q0.x, q1.x, q0.y, q1.y}, hi[4] = {q0.z, q1.z, q0.w, q1.w};
                    #pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        mma_s8_16832(acc[i][n], lo, b[k][n].x, b[k][n].y);
                        mma_s8_16832(acc[i][n], hi, b[k][n].z, b[k][n].w);
                    }
                }
            }
            if (NP <= 2 && st + 1 < stages) load_b(st + 1);
        }
        if (Up<NP>::kParities == 1) sync_worker();  // the sums before have been taken
        const auto put_sums = [&](bool add) {
            #pragma unroll
            for (int i = 0; i < TILES; ++i) {
                #pragma unroll
                for (int n = 0; n < NP; ++n) {
                    #pragma unroll
                    for (int c = 0; c < 4; c += 2) {
                        int2* const to = reinterpret_cast<int2*>(
                            &sums[parity][PAIRED ? (warp & 1) + 2 * i : warp][g + 4 * c][8 * n + 2 * t]);
                        const int2 had = add ? *to : make_int2(0, 0);
                        *to = make_int2(had.x + acc[i][n][c], had.y + acc[i][n][c + 1]);
                    }
                }
            }
        };
        if (!PAIRED || warp < 2) put_sums(false);
        if constexpr (PAIRED) {
            sync_worker();
            if (warp >= 2) put_sums(true);
        }
        sync_worker();
        // Warp j: the job's tokens j, j + 4; lane: one of the 32 rows. (A
        // barrier of the next item comes before these sums are written again.)
        for (int j = warp; j < job.count; j += kUpWarps) {
            const int m = r.token[job.pos + j];
            const int h2 = item % halves;
            const int run = lane >> 3, f = h2 / 2 * 64 + 16 * run + 8 * (h2 & 1) + (lane & 7);
            const int tile = run >> 1, row = 8 * (run & 1) + (lane & 7);
            const float unit = a.xs[m];
            const int64_t at = static_cast<int64_t>(job.expert) * a.F + min(f, a.F - 1);
            const float sg = a.sg[at], su = a.su[at];
            const auto dot = [&](const int (&s)[16][8 * NP]) {
                const int4 d = *reinterpret_cast<const int4*>(&s[row][4 * j]);
                return static_cast<float>(((static_cast<double>(d.w) * 256.0 + d.z) * 256.0 + d.y) * 256.0 + d.x);
            };
            const float gv = dot(sums[parity][tile]) * unit * sg, uv = dot(sums[parity][2 + tile]) * unit * su;
            const float h = f < a.F ? gv / (1.0f + expf(-gv)) * uv : 0.0f;
            const bool bad = __any_sync(0xffffffffu, not_finite(h));
            const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(h))));
            const Fixed fx = fixed_for(top, bad);
            const uint32_t y = bad ? 0u : digits_of(h, fx);
            const int64_t pair = r.pair[job.pos + j];
            int8_t* hd = a.hd + pair * 4 * a.fp + f;
            #pragma unroll
            for (int i = 0; i < 4; ++i) hd[static_cast<int64_t>(i) * a.fp] = static_cast<int8_t>(y >> (8 * i));
            if (lane == 0) a.hs[pair * (a.fp / 32) + h2] = fx.unit;
        }
    }
    cp_async_wait_group<0>();
}

// -------------------------------------------------------------------- down
// A block is an SM's whole load, 16 warps, and owns `rows` (at most 8 GROUPS)
// output channels at a time: 14 for 2048 channels, 18 for 2560. Its warps share
// the (job, stage) list of a tile in equal runs, so that no other block is needed
// for a token's sum over its experts; they stream it, from one tile into the
// next, through rings in shared memory. A step's exact integer sums join in f32
// with the step's unit. At the end of a job a warp adds its result, weighted, to
// its own sums per token; the warps' are added in order at the end of the tile.
//
// Every tile reads all digits of the hidden values (4 bytes a value, from L2), so
// with several tokens to an expert a tile has up to 32 rows, two M sides that
// share them: 2560 channels as 18 rows a tile instead of twice 9 took 55 us
// instead of 71 (24 picks among 24 experts of 5056), 197 instead of 380 (25
// tokens that all pick all 8 experts of 6448), 4096 as 28 instead of twice 14 43
// instead of 49 (72 picks among 64 of 1088). One token's are few: it stays with
// the 16-row tiles, whose copies take 256 bytes of a row at a time.
template <int NP, int GROUPS>
struct Down {
    static constexpr int kRows = 8 * GROUPS;
    static constexpr int kTiles = (GROUPS + 1) / 2;           // M sides
    static constexpr int kWide = GROUPS == 2 && NP < 4 ? 4 : 2;  // windows of a stage, what registers allow
    static constexpr int kCols = 64 * kWide;
    static constexpr int kBytes = 512 * GROUPS * kWide;       // of a stage: [window][row][64 bytes]
    static constexpr int bytes(int stages, int tokens) {      // of shared memory
        return kDownWarps * (stages * kBytes + tokens * kRows * static_cast<int>(sizeof(float)));
    }
};

template <int NP, int GROUPS, int STAGES>
__global__ void __launch_bounds__(kDownThreads, 1) down_kernel(const MoeArgs a) {
    using D = Down<NP, GROUPS>;
    constexpr int TILES = D::kTiles, WIDE = D::kWide, ROWS = D::kRows;
    extern __shared__ __align__(128) uint8_t s_raw[];
    float* const outs = reinterpret_cast<float*>(s_raw + kDownWarps * STAGES * D::kBytes);  // [warp][token][ROWS]
    __shared__ Routing r;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    pdl_launch_dependents();
    for (int i = tid; i < kDownWarps * a.M * ROWS; i += kDownThreads) outs[i] = 0.0f;
    pdl_wait();
    for (int i = tid; i < a.M * a.top; i += kDownThreads) {
        r.pick[i] = static_cast<short>(a.experts[i]);
        r.weight[i] = a.weights[i];
    }
    __syncthreads();
    list_jobs<NP, kDownThreads>(a, r);

    const int stages = a.fp / D::kCols, tiles = (a.K + a.rows - 1) / a.rows;
    const int units = r.jobs * stages;  // under 2^19
    const int u_begin = units * warp / kDownWarps, u_end = units * (warp + 1) / kDownWarps;
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(s_raw)) + warp * STAGES * D::kBytes + 16 * lane;
    float* const mine = outs + warp * a.M * ROWS;

    // The copying side: tile, job, stage of it, this lane's rows g, g + 8, ...
    int c_tile = blockIdx.x, c_left = u_end - u_begin, c_job = u_begin / stages, c_s = u_begin % stages, c_slot = 0;
    int bytes[GROUPS] = {};
    const int8_t* rows[GROUPS] = {};
    const auto rows_of = [&] {
        const int n0 = c_tile * a.rows, n_end = min(a.K, n0 + a.rows);
        const int64_t at = static_cast<int64_t>(job_of(r, c_job).expert) * a.K;
        #pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            bytes[i] = n0 + 8 * i + g < n_end ? 16 : 0;
            rows[i] = a.qd + (at + min(n0 + 8 * i + g, a.K - 1)) * a.F + 16 * t;
        }
    };
    const auto copy_next = [&] {
        if (c_left > 0) {
            copy_stage<GROUPS, WIDE>(ring + c_slot * D::kBytes, rows, bytes, c_s * D::kCols, t, a.F);
            --c_left;
            ++c_s;
            if (c_left == 0) {
                c_tile += gridDim.x;
                c_job = u_begin / stages, c_s = u_begin % stages;
                if (c_tile < tiles) c_left = u_end - u_begin, rows_of();
            } else if (c_s == stages) {
                c_s = 0;
                ++c_job;
                rows_of();
            }
        }
        cp_async_commit();
        c_slot = c_slot == STAGES - 1 ? 0 : c_slot + 1;
    };
    if (c_left > 0) rows_of();
    #pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) copy_next();

    int slot = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int n0 = tile * a.rows, n_end = min(a.K, n0 + a.rows);
        for (int u = u_begin; u < u_end;) {
            const int s_begin = u % stages;
            const Job job = job_of(r, u / stages);
            const int s_end = min(stages, s_begin + (u_end - u));
            u += s_end - s_begin;
            // This lane's column of the B operand, and the token of its result
            // columns (columns of tokens that the job does not have are not used).
            const int8_t* hd[NP];
            const float* hs[NP];
            #pragma unroll
            for (int n = 0; n < NP; ++n) {
                const int j = min(2 * n + (g >> 2), job.count - 1), jr = min(2 * n + (t >> 1), job.count - 1);
                hd[n] = a.hd + (static_cast<int64_t>(r.pair[job.pos + j]) * 4 + (g & 3)) * a.fp + 16 * t;
                hs[n] = a.hs + static_cast<int64_t>(r.pair[job.pos + jr]) * (a.fp / 32);
            }
            float scale[GROUPS];
            #pragma unroll
            for (int i = 0; i < GROUPS; ++i) {
                scale[i] = a.sd[static_cast<int64_t>(job.expert) * a.K + min(n0 + 8 * i + g, n_end - 1)];
            }
            uint4 b[WIDE][NP];
            float2 unit[WIDE][NP];
            const auto load_b = [&](int st) {
                #pragma unroll
                for (int n = 0; n < NP; ++n) {
                    #pragma unroll
                    for (int k = 0; k < WIDE; ++k) {
                        b[k][n] = *reinterpret_cast<const uint4*>(hd[n] + D::kCols * st + 64 * k);
                    }
                    #pragma unroll
                    for (int k = 0; k < WIDE; k += 2) {
                        const float4 x = *reinterpret_cast<const float4*>(hs[n] + 2 * WIDE * st + 2 * k);
                        unit[k][n] = make_float2(x.x, x.y), unit[k + 1][n] = make_float2(x.z, x.w);
                    }
                }
            };
            if (NP == 1) load_b(s_begin);
            float2 acc2[TILES][NP][2] = {};
            for (int st = s_begin; st < s_end; ++st) {
                if (NP > 1) load_b(st);  // (too many registers to hold a stage ahead)
                cp_async_wait_group<STAGES - 2>();
                __syncwarp();
                copy_next();
                const uint32_t at = ring + slot * D::kBytes;
                slot = slot == STAGES - 1 ? 0 : slot + 1;
                #pragma unroll
                for (int k = 0; k < WIDE; ++k) {
                    #pragma unroll
                    for (int i = 0; i < TILES; ++i) {
                        const uint32_t from = at + 512 * (GROUPS * k + 2 * i);
                        const uint4 q0 = load_shared16(from);
                        const uint4 q1 = 2 * i + 1 < GROUPS ? load_shared16(from + 512) : make_uint4(0, 0, 0, 0);
                        const uint32_t lo[4] = {q0.x, q1.x, q0.y, q1.y}, hi[4] = {q0.z, q1.z, q0.w, q1.w};
                        #pragma unroll
                        for (int n = 0; n < NP; ++n) {
                            int d[2][4];
                            mma_s8_16832_from(d[0], lo, b[k][n].x, b[k][n].y, kMagicBits);
                            mma_s8_16832_from(d[1], hi, b[k][n].z, b[k][n].w, kMagicBits);
                            #pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const float by = h == 0 ? unit[k][n].x : unit[k][n].y;
                                #pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    if (2 * i + c >= GROUPS) continue;
                                    const float2 x = __fadd2_rn(make_float2(__int_as_float(d[h][2 * c]), __int_as_float(d[h][2 * c + 1])),
                                                                make_float2(-kMagic, -kMagic));
                                    acc2[i][n][c] = __ffma2_rn(x, make_float2(by, by), acc2[i][n][c]);
                                }
                            }
                        }
                    }
                }
                if (NP == 1 && st + 1 < s_end) load_b(st + 1);
            }
            #pragma unroll
            for (int n = 0; n < NP; ++n) {
                // Lane (g, t) has digits 2 (t % 2) and 2 (t % 2) + 1 of token t / 2.
                const int j = 2 * n + (t >> 1);
                #pragma unroll
                for (int i = 0; i < GROUPS; ++i) {
                    const float2 d = acc2[i / 2][n][i % 2];
                    float v = fmaf(d.y, 256.0f, d.x);
                    v = fmaf(__shfl_xor_sync(0xffffffffu, v, 1), (t & 1) ? 0.0f : 65536.0f, v);
                    if (j < job.count && !(t & 1)) {
                        mine[r.token[job.pos + j] * ROWS + 8 * i + g] += v * scale[i] * r.weight[r.pair[job.pos + j]];
                    }
                }
            }
        }
        __syncthreads();
        for (int i = tid; i < a.M * ROWS; i += kDownThreads) {
            const int m = i / ROWS, n = n0 + i % ROWS;
            float v = 0.0f;
            #pragma unroll
            for (int w = 0; w < kDownWarps; ++w) {
                v += outs[w * a.M * ROWS + i];
                outs[w * a.M * ROWS + i] = 0.0f;
            }
            if (n < n_end) a.out[static_cast<int64_t>(m) * a.K + n] = v;
        }
        __syncthreads();
    }
    cp_async_wait_group<0>();
}

// --------------------------------------------------- any sizes and alignment
// Sizes that are not multiples of 16 and unaligned codes: one warp per value.
__global__ void __launch_bounds__(kMoeThreads) plain_up_kernel(const MoeArgs a) {
    __shared__ Routing r;
    pdl_launch_dependents();
    pdl_wait();
    route_tokens<kMoeThreads>(a, r);
    const int lane = threadIdx.x & 31;
    const int64_t total = static_cast<int64_t>(a.M) * a.top * a.F;
    for (int64_t i = blockIdx.x * kMoeWarps + (threadIdx.x >> 5); i < total; i += gridDim.x * kMoeWarps) {
        const int pair = static_cast<int>(i / a.F), f = static_cast<int>(i % a.F);
        const int64_t at = static_cast<int64_t>(r.pick[pair]) * a.F + f;
        const float* x = a.x + static_cast<int64_t>(pair / a.top) * a.K;
        float g = 0.0f, u = 0.0f;
        for (int k = lane; k < a.K; k += 32) {
            g = fmaf(x[k], static_cast<float>(a.qg[at * a.K + k]), g);
            u = fmaf(x[k], static_cast<float>(a.qu[at * a.K + k]), u);
        }
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            g += __shfl_xor_sync(0xffffffffu, g, o);
            u += __shfl_xor_sync(0xffffffffu, u, o);
        }
        g *= a.sg[at];
        if (lane == 0) a.h[i] = g / (1.0f + expf(-g)) * (u * a.su[at]);
    }
}

__global__ void __launch_bounds__(kMoeThreads) plain_down_kernel(const MoeArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t total = static_cast<int64_t>(a.M) * a.K;
    for (int64_t i = blockIdx.x * kMoeWarps + (threadIdx.x >> 5); i < total; i += gridDim.x * kMoeWarps) {
        const int m = static_cast<int>(i / a.K), n = static_cast<int>(i % a.K);
        float out = 0.0f;
        for (int j = 0; j < a.top; ++j) {
            const int pair = m * a.top + j;
            const int64_t at = static_cast<int64_t>(a.experts[pair]) * a.K + n;
            float v = 0.0f;
            for (int f = lane; f < a.F; f += 32) {
                v = fmaf(a.h[static_cast<int64_t>(pair) * a.F + f], static_cast<float>(a.qd[at * a.F + f]), v);
            }
            #pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            out = fmaf(v * a.sd[at], a.weights[pair], out);
        }
        if (lane == 0) a.out[i] = out;
    }
}

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

bool sizes_supported(int64_t M, int64_t K, int64_t F, int64_t E, int64_t top) {
    // 65536 columns keep a digit's sum inside 31 bits.
    return K <= 65536 && F <= 65536 && E <= kMoeExperts && top <= kMoeTop && top <= E && M <= (int64_t{1} << 30);
}

// Whether the tensor kernels take these sizes (alignment aside).
bool tensor_sizes(int64_t K, int64_t F) { return K % 16 == 0 && F % 16 == 0; }

// Places of the scratch buffers; returns the bytes they take.
int64_t lay_out(MoeArgs& a, char* ws, int64_t M, bool tensor, bool own_picks) {
    int64_t at = 0;
    const auto take = [&](int64_t bytes) {
        char* p = ws + at;
        at += round_up(bytes, 256);
        return p;
    };
    const int64_t pairs = M * a.top;
    a.logits = reinterpret_cast<float*>(take(4 * M * a.E));
    int* const experts = reinterpret_cast<int*>(take(4 * pairs));
    float* const weights = reinterpret_cast<float*>(take(4 * pairs));
    if (own_picks) a.experts = experts, a.weights = weights;
    if (tensor) {
        a.xd = reinterpret_cast<int8_t*>(take(M * 4 * a.kp));
        a.xs = reinterpret_cast<float*>(take(4 * M));
        a.hd = reinterpret_cast<int8_t*>(take(pairs * 4 * a.fp));
        a.hs = reinterpret_cast<float*>(take(pairs * (a.fp / 32) * 4));
    } else {
        a.h = reinterpret_cast<float*>(take(4 * pairs * a.F));
    }
    return at;
}

// Lets a kernel have BYTES of shared memory, once for each device. (The same
// number from every call: threads that get here together set the same limit.)
template <int BYTES, class Kernel>
cudaError_t allow_shared(Kernel kernel, bool (&allowed)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 64 && __atomic_load_n(&allowed[dev], __ATOMIC_RELAXED)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
    if (e == cudaSuccess && dev < 64) __atomic_store_n(&allowed[dev], true, __ATOMIC_RELAXED);
    return e;
}

template <int NP, int GROUPS, int STAGES>
cudaError_t run_down(const MoeArgs& a, int blocks, cudaStream_t stream) {
    const int bytes = Down<NP, GROUPS>::bytes(STAGES, a.M);  // at most kDownShared (run_down_sized)
    static bool allowed[64] = {};
    const cudaError_t e = allow_shared<kDownShared>(down_kernel<NP, GROUPS, STAGES>, allowed);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg =
        pdl_config(dim3(static_cast<unsigned>(blocks)), dim3(kDownThreads), static_cast<size_t>(bytes), stream, attr);
    return cudaLaunchKernelEx(&cfg, down_kernel<NP, GROUPS, STAGES>, a);
}

// As many tiles for every SM, as few as `most` rows a tile allow.
int tile_rows(int K, int most, int64_t sms) { return static_cast<int>(ceil_div(K, ceil_div(K, most * sms) * sms)); }

template <int NP>
cudaError_t run_down_sized(MoeArgs a, cudaStream_t stream) {
    const int64_t sms = device_sm_count();
    a.rows = tile_rows(a.K, 16, sms);
    const auto blocks = [&] { return static_cast<int>(std::min(ceil_div(a.K, a.rows), sms)); };
    if constexpr (NP > 1) {
        const int rows = tile_rows(a.K, 32, sms);
        MoeArgs wide = a;
        wide.rows = rows;
        const int at = static_cast<int>(std::min(ceil_div(a.K, rows), sms));
        if (rows > 24 && Down<NP, 4>::bytes(2, a.M) <= kDownShared) {
            return Down<NP, 4>::bytes(3, a.M) <= kDownShared ? run_down<NP, 4, 3>(wide, at, stream)
                                                         : run_down<NP, 4, 2>(wide, at, stream);
        }
        if (rows > 16 && rows <= 24 && Down<NP, 3>::bytes(3, a.M) <= kDownShared) {
            return Down<NP, 3>::bytes(4, a.M) <= kDownShared ? run_down<NP, 3, 4>(wide, at, stream)
                                                         : run_down<NP, 3, 3>(wide, at, stream);
        }
    }
    constexpr int HALF = Down<NP, 2>::kWide == 4 ? 1 : 2;  // stages of half the size
    return Down<NP, 2>::bytes(3 * HALF, a.M) <= kDownShared ? run_down<NP, 2, 3 * HALF>(a, blocks(), stream)
                                                            : run_down<NP, 2, 2 * HALF>(a, blocks(), stream);
}

template <int NP>
cudaError_t run_tensor(MoeArgs a, cudaStream_t stream) {
    const int64_t sms = device_sm_count();
    static bool allowed[64] = {};
    cudaError_t e = allow_shared<Up<NP>::kBytes>(up_kernel<NP>, allowed);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    const int64_t items = static_cast<int64_t>(a.M) * a.top * ((a.F + 63) / 64 * 2);  // at most
    const cudaLaunchConfig_t cfg = pdl_config(dim3(static_cast<unsigned>(items < sms ? items : sms)),
                                              dim3(kUpWorkers * kUpThreads), Up<NP>::kBytes, stream, attr);
    e = cudaLaunchKernelEx(&cfg, up_kernel<NP>, a);
    if (e != cudaSuccess) return e;
    return run_down_sized<NP>(a, stream);
}

cudaError_t run_pass(const MoeArgs& a, bool tensor, cudaStream_t stream) {
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = pdl_config(dim3(a.E + (tensor ? a.M : 0), (a.M + 7) / 8), dim3(kRouteThreads), 0,
                                        stream, attr);
    cudaError_t e = cudaLaunchKernelEx(&cfg, route_kernel, a);
    if (e != cudaSuccess) return e;
    if (!tensor) {
        cfg.gridDim = dim3(4 * device_sm_count());
        cfg.blockDim = dim3(kMoeThreads);
        e = cudaLaunchKernelEx(&cfg, plain_up_kernel, a);
        return e != cudaSuccess ? e : cudaLaunchKernelEx(&cfg, plain_down_kernel, a);
    }
    // Tokens of a job: two, four or eight. One or two tokens rarely share an expert
    // (2 tokens, 2 of 16 experts of 4096 x 11008: 92 us with two, 103 with four). A
    // job of eight costs more than one of four and pays where most experts have more
    // than four tokens: 24, 32 and 40 tokens, 2 of 16 experts of 4096 x 5504, 201,
    // 243 and 293 us with four, 228, 250 and 258 with eight; 11, 32 and 64 tokens, 6
    // of 64 of 2048 x 1424, 84, 133 and 200 against 104, 149 and 189; 4 and 5 tokens
    // on all of 8 of 2560 x 2576, 52 and 69 against 66 and 67.
    if (a.M <= 2) return run_tensor<1>(a, stream);
    if (a.M * a.top <= 4 * a.E) return run_tensor<2>(a, stream);
    return run_tensor<4>(a, stream);
}

}  // namespace
}  // namespace pcb

extern "C" int64_t popcornMoeWorkspace(int64_t M, int64_t K, int64_t F, int64_t E, int64_t top_k) {
    if (M <= 0 || K <= 0 || F <= 0 || E <= 0 || top_k <= 0 || !pcb::sizes_supported(M, K, F, E, top_k)) return 0;
    pcb::MoeArgs a = {};
    a.K = static_cast<int>(K), a.F = static_cast<int>(F), a.E = static_cast<int>(E), a.top = static_cast<int>(top_k);
    a.kp = static_cast<int>(pcb::round_up(K, pcb::kColumns)), a.fp = static_cast<int>(pcb::round_up(F, pcb::kColumns));
    const int64_t m = M < pcb::kMoeTokens ? M : pcb::kMoeTokens;
    // (Either kind of kernel: the sizes do not say how the codes are aligned.)
    const int64_t plain = pcb::lay_out(a, nullptr, m, false, true);
    const int64_t tensor = pcb::tensor_sizes(K, F) ? pcb::lay_out(a, nullptr, m, true, true) : 0;
    return plain > tensor ? plain : tensor;
}

extern "C" popcornStatus_t popcornMoe_i8f32(float* out, int32_t* experts, float* weights, const float* x,
                                            const float* router, const int8_t* q_gate, const float* s_gate,
                                            const int8_t* q_up, const float* s_up, const int8_t* q_down,
                                            const float* s_down, int64_t M, int64_t K, int64_t F, int64_t E,
                                            int64_t top_k, int renormalize, void* workspace, int64_t workspace_bytes,
                                            cudaStream_t stream) {
    if (out == nullptr || x == nullptr || router == nullptr || q_gate == nullptr || s_gate == nullptr ||
        q_up == nullptr || s_up == nullptr || q_down == nullptr || s_down == nullptr ||
        (experts == nullptr) != (weights == nullptr)) {
        return POPCORN_ERROR_INVALID_VALUE;
    }
    if (M <= 0 || K <= 0 || F <= 0 || E <= 0) return POPCORN_SUCCESS;
    if (top_k <= 0 || !pcb::sizes_supported(M, K, F, E, top_k)) return POPCORN_ERROR_INVALID_VALUE;
    const int64_t need = popcornMoeWorkspace(M, K, F, E, top_k);
    void* ws = workspace;
    if (workspace == nullptr) {
        const cudaError_t e = pcb::scratch_alloc(&ws, static_cast<size_t>(need), stream);
        if (e != cudaSuccess) return pcb::record_cuda(e);
    } else if (workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) {
        return POPCORN_ERROR_INVALID_VALUE;
    }
    const bool tensor = pcb::tensor_sizes(K, F) && pcb::aligned16(q_gate) && pcb::aligned16(q_up) && pcb::aligned16(q_down);
    pcb::MoeArgs a = {};
    a.router = router, a.qg = q_gate, a.sg = s_gate, a.qu = q_up, a.su = s_up, a.qd = q_down, a.sd = s_down;
    a.K = static_cast<int>(K), a.F = static_cast<int>(F), a.E = static_cast<int>(E), a.top = static_cast<int>(top_k);
    a.renorm = renormalize;
    a.kp = static_cast<int>(pcb::round_up(K, pcb::kColumns)), a.fp = static_cast<int>(pcb::round_up(F, pcb::kColumns));
    cudaError_t e = cudaSuccess;
    for (int64_t m = 0; m < M && e == cudaSuccess; m += pcb::kMoeTokens) {
        a.M = static_cast<int>(M - m < pcb::kMoeTokens ? M - m : pcb::kMoeTokens);
        a.out = out + m * K, a.x = x + m * K;
        if (experts != nullptr) a.experts = experts + m * top_k, a.weights = weights + m * top_k;
        pcb::lay_out(a, static_cast<char*>(ws), M < pcb::kMoeTokens ? M : pcb::kMoeTokens, tensor, experts == nullptr);
        e = pcb::run_pass(a, tensor, stream);
    }
    if (workspace == nullptr) {
        const cudaError_t f = pcb::scratch_free(ws, stream);
        if (e == cudaSuccess) e = f;
    }
    if (e != cudaSuccess) return pcb::record_cuda(e);
    return pcb::check_launch();
}
