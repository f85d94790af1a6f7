// Attention over the paged 8-bit key/value cache.
//
// out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max),  with
// k_j = ck_j ks, v_j = cv_j vs: codes ck, cv and one scale for each block of
// a page's tokens and a head. The block scales leave the inner products:
// q . k_j = (q . ck_j) ks, and vs joins p_j.
//
// Few query rows (kv_rows_kernel). What it cannot do without is one read of
// the visible codes, 2 dim bytes a token and head; it is bound by HBM. Layout:
//  * A warp takes 16 tokens at a time. Tokens are the M side of the matrix
//    instructions and up to 8 NT query rows (the heads that share a key head,
//    times the sequence's tokens) their N side, so that a few rows fill the
//    instruction better than with queries as M. The operands of both products
//    are read in 16-byte pieces: the sums over dim and over tokens may run in
//    any order, so each lane takes whole pieces and the other operand is
//    permuted to match.
//  * Every warp streams its tiles through a ring of its own in shared memory by
//    16-byte asynchronous copies, two to seven tiles ahead, without barriers.
//    (Loads into registers kept 4 KB a warp in flight, 64 KB an SM: 102 us for
//    64 ragged sequences, bf16, against 87 us.)
//  * Scores: mma s8 x s8 -> s32 on the raw key codes; each query row is fixed
//    point in signed base-256 digits (2 for f16 / bf16, 3 for f32), each
//    digit one product, so the sums are exact integers. The accumulators
//    start at the bits of 1.5 2^23, which makes them floats at no cost.
//  * Softmax: running maximum m of log2-domain scores plus the exponent of vs
//    (so that p vs stays in range whatever the scales are); it moves only when
//    a score exceeds it by 2^8, which is rare after the first tiles, so most
//    tiles pay one vote instead of a reduction. Probabilities are scaled by
//    2^6 to keep small ones out of f16's subnormals (largest 2^15).
//  * Values: codes become f16 exactly (byte permutes), probabilities f16 for
//    bf16 outputs and f16 high + f16 rest for f16 and f32, products accumulate
//    in f32. For f32 each tile's product starts from zero and is added to the
//    running sum by an ordinary f32 add: the tensor cores' accumulation
//    truncates, which over hundreds of tiles costs more than f32 should lose.
//  * Tasks of 16-token tiles, cut over the workers of all SMs
//    (kv_attention.cuh); split tasks are joined by kv_join_kernel.
//
// Measured, with the join, in a graph: 16 sequences of 4096 tokens, 32 key heads of
// 128, one f32 query each: 99 us, 5.4 TB/s; 64 ragged ones up to 8192, 8 key heads,
// bf16: 87 us, 5.7 TB/s; one of 131,075 tokens, f16: 55 us, 4.9 TB/s. Small calls
// are a chain of latencies (schedule, block table, codes, partial results, join):
// 12 us for 1000 tokens. Ragged batches of short sequences are far from HBM's rate:
// below 4 kTaskUnits tiles a worker the runs are equal in tiles, however many tasks
// they hold (64 sequences up to 512, 32 heads, f16: 204 us, floor 21).
//
// Sequences with many query rows go to the kernel of kv_prompt.cu where it takes
// their type and dim (kPromptRows).
#include <algorithm>
#include <type_traits>

#include "kv_attention.cuh"
#include "mma_frag.cuh"

namespace pcb {
namespace {

__device__ unsigned int g_attn_err = 0;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr float kMagic = 12582912.0f;       // 1.5 2^23
constexpr int kMagicBits = 0x4B400000;
constexpr int kTaskUnits = 24;             // a task's fixed cost in tiles (5 us: its queries, its first tiles, its join)

// d = c + a b with all of c the same value (mma_frag.cuh has the s8 form).
__device__ __forceinline__ void mma_f16_16816_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                                   float c) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c));
}

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Transposes the warp's 8 x 8 matrix of 16-bit elements.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Two f16 of signed codes from the biased bytes (code + 128) that `sel` picks
// out of w: byte u in the low mantissa byte of 1024 is 1024 + u.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
    const uint32_t x = __byte_perm(w, 0x64646464u, SEL);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2{__float2half_rn(1152.0f), __float2half_rn(1152.0f)});
    return *reinterpret_cast<const uint32_t*>(&h);
}

// A lane's part of a query row: lane (g, t) = (lane / 4, lane % 4) holds, of
// row g, the 16-byte pieces t, t + 4, ... of dim that lane (., t) reads of a
// key.
template <typename T, int DP>
struct Query {
    alignas(16) T v[DP / 64][16];
};
template <typename T, int DP>
__device__ __forceinline__ void load_query(Query<T, DP>& q, const T* row, bool valid, int dim, bool vec, int t) {
    #pragma unroll
    for (int c = 0; c < DP / 64; ++c) {
        const int d0 = 16 * (t + 4 * c);
        const bool in = valid && d0 < dim;
        #pragma unroll
        for (int w = 0; w < 16; w += 4) {
            if (in && vec) {
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<float4*>(&q.v[c][w]) = *reinterpret_cast<const float4*>(row + d0 + w);
                } else {
                    *reinterpret_cast<uint2*>(&q.v[c][w]) = *reinterpret_cast<const uint2*>(row + d0 + w);
                }
            } else {
                #pragma unroll
                for (int j = 0; j < 4; ++j) q.v[c][w + j] = in ? row[d0 + w + j] : from_f32<T>(0.0f);
            }
        }
    }
}

// The row as the B operand of the score products: DIGITS words for each
// 32-wide step's two halves, and the row's factor.
template <typename T, int DP, int DIGITS>
__device__ __forceinline__ float query_digits(uint32_t (&qd)[DIGITS][DP / 16], const Query<T, DP>& q) {
    constexpr int PIECES = DP / 64;
    float m = 0.0f;
    bool bad = false;
    #pragma unroll
    for (int c = 0; c < PIECES; ++c) {
        #pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float v = fabsf(to_f32(q.v[c][j]));
            m = fmaxf(m, v);
            bad = bad || !(v <= 3.4028234663852886e38f);
        }
    }
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    int nan = bad;
    nan |= __shfl_xor_sync(0xffffffffu, nan, 1);
    nan |= __shfl_xor_sync(0xffffffffu, nan, 2);
    // Three digits: a power of two that brings the largest element to
    // [2^21, 2^22), exact and inside the balanced digits' range. Two digits:
    // the largest element becomes 32512 = 127 * 256, since with a power of two
    // the 15 bits could be too few for f16 queries' 11.
    float up, down;
    if constexpr (DIGITS == 3) {
        const int e = max(-126, min(120, 21 + 127 - static_cast<int>(__float_as_uint(m) >> 23)));
        up = __int_as_float((127 + e) << 23);
        down = __int_as_float((127 - e) << 23);
    } else {
        const float most = fmaxf(m, 1e-30f);
        up = 32512.0f / most;
        down = most / 32512.0f;
    }
    constexpr uint32_t BIAS = DIGITS == 2 ? 0x8080u : 0x808080u;
    #pragma unroll
    for (int c = 0; c < PIECES; ++c) {
        #pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t y[4];
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float v = nan ? 0.0f : to_f32(q.v[c][4 * w + j]);
                y[j] = static_cast<uint32_t>(__float2int_rn(v * up)) + BIAS;
            }
            #pragma unroll
            for (int i = 0; i < DIGITS; ++i) {
                const uint32_t sel = static_cast<uint32_t>(i | ((i + 4) << 4));
                qd[i][4 * c + w] =
                    __byte_perm(__byte_perm(y[0], y[1], sel), __byte_perm(y[2], y[3], sel), 0x5410) ^ 0x80808080u;
            }
        }
    }
    return nan ? __int_as_float(0x7fffffff) : down;
}

template <typename T>
struct Traits {
    static constexpr int kDigits = 2;     // of a query element
    static constexpr bool kSplit = false; // probabilities as two f16
    static constexpr bool kFresh = false; // each tile's product summed on its own
};
template <>
struct Traits<__half> {
    static constexpr int kDigits = 2;
    static constexpr bool kSplit = true;  // one f16 would add as much error as f16 outputs have
    static constexpr bool kFresh = false;
};
template <>
struct Traits<float> {
    static constexpr int kDigits = 3;
    static constexpr bool kSplit = true;
    static constexpr bool kFresh = true;
};

// A block of kv_rows_kernel is an SM's whole load: as many workers of four
// warps as its registers hold, each with its own run and barrier, and each warp
// with a ring of tiles in shared memory, 16 rows of keys and 16 of values a
// tile. The rings take 192 KB, most of it in flight, which is what it takes to
// stream at HBM's rate. (Workers as blocks of their own, three to an SM, left
// holes in the registers where they met the blocks of another kernel: the
// one that did not fit began when others ended, 69 us against 55 for 131075
// tokens, f16.)
template <typename T, int DP, int NT>
struct Rows {
    static constexpr int kWorkers = DP == 256 ? 2 : 3;
    static constexpr int kTileBytes = 2 * 16 * DP;
    static constexpr int kStages = (192 / kWorkers) * 1024 / (kWarps * kTileBytes);  // 3 to 8
    static constexpr int kRing = kWarps * kStages * kTileBytes;                      // of a worker
    static constexpr int kScales = kWorkers * kRing;                                 // [warp][stage] {ks, vs}
    static constexpr int kBytes = kScales + kWorkers * kWarps * kStages * 8;
    static_assert(kRing >= kWarps * 8 * NT * DP * 4, "the warps' sums take the ring's place");
};

__device__ __forceinline__ void load_shared(uint32_t (&w)[4], uint32_t addr) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(addr));
}
__device__ __forceinline__ void load_shared(uint32_t (&w)[2], uint32_t addr) {
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
}

// DP: dim rounded up to 64, 128 or 256; FULL: dim is DP.
template <typename T, int DP, int NT, bool FULL>
__global__ void __launch_bounds__((kThreads * Rows<T, DP, NT>::kWorkers), 1) kv_rows_kernel(const AttnArgs a) {
    using R = Rows<T, DP, NT>;
    constexpr int DIGITS = Traits<T>::kDigits;
    constexpr bool SPLIT = Traits<T>::kSplit, FRESH = Traits<T>::kFresh;
    constexpr int ROWS = 8 * NT;
    constexpr int STAGES = R::kStages;
    constexpr int CH = DP / 16;                // 16-byte pieces of a row
    constexpr int KP = DP / 64;                // ... of a key row per lane
    constexpr int VW = DP == 64 ? 2 : 4;       // words per piece of a value row
    constexpr int VP = DP == 256 ? 2 : 1;      // pieces of a value row per lane
    constexpr int NJ = DP / 16;                // 16-wide steps of dim in the value product
    constexpr int COPIES = CH / 2;             // 16-byte copies of a lane for 16 rows
    __shared__ float s_mls[R::kWorkers][kWarps][ROWS][2];
    extern __shared__ __align__(128) uint8_t s_ring[];
    const int worker = threadIdx.x / kThreads;  // of the block
    float (*const s_o)[ROWS][DP] = reinterpret_cast<float (*)[ROWS][DP]>(s_ring + worker * R::kRing);  // after a task's tiles
    float (*const s_ml)[ROWS][2] = s_mls[worker];
    const auto sync_worker = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1 + worker), "n"(kThreads) : "memory"); };

    const uint32_t smem_ring = static_cast<uint32_t>(__cvta_generic_to_shared(s_ring));
    const int dim = FULL ? DP : a.dim;
    const int tid = threadIdx.x % kThreads, lane = tid & 31, warp = tid >> 5;  // of the worker
    const int g = lane >> 2, t = lane & 3;
    pdl_launch_dependents();
    pdl_wait();

    // A sequence's tiles are those that its first and last query see together.
    const auto tiles_of = [&](const Seq& s, Span& see) {
        see = span_of(a, s, 0, s.rows - 1);
        return (see.hi - see.lo + 15) >> 4;
    };
    // Worker g gridDim.x + blockIdx.x: the first ones of all blocks before the second.
    const Run run = find_run<true>(a.seqs, worker * gridDim.x + blockIdx.x, R::kWorkers * gridDim.x, kWarps, kTaskUnits, [&](int b, int64_t& tiles, int64_t& tasks) {
        const Seq s = sequence(a, b, &g_attn_err);
        Span see;
        tasks = static_cast<int64_t>((s.rows * a.group + ROWS - 1) / ROWS) * a.heads;
        tiles = tasks * max(tiles_of(s, see), 1);
    });
    if (tid == 0) clear_entries(a, run);
    int64_t run0 = run.begin, from = run.from, task0 = run.task0;
    int b = run.b;

    while (run0 < run.end) {
        const Seq s = sequence(a, b, &g_attn_err);
        Span see;
        const int seen_tiles = tiles_of(s, see), tiles = max(seen_tiles, 1);
        const int row_tiles = (s.rows * a.group + ROWS - 1) / ROWS;
        const int pieces = run.piece ? static_cast<int>(divide(tiles + run.piece - 1, run.piece)) : 1;
        const int each = run.piece ? pieces : run.fixed + tiles;
        const int64_t units = static_cast<int64_t>(row_tiles) * a.heads * each;
        if (run0 >= from + units) {
            from += units;
            task0 += static_cast<int64_t>(row_tiles) * a.heads;
            ++b;
            continue;
        }
        const int task = static_cast<int>(divide(run0 - from, each));
        const int c0 = static_cast<int>(run0 - from - static_cast<int64_t>(task) * each);
        const int c1 = static_cast<int>(min(static_cast<int64_t>(each), c0 + (run.end - run0)));
        run0 += c1 - c0;
        int u0, u1;
        if (run.piece) {
            u0 = static_cast<int>(divide(static_cast<int64_t>(tiles) * c0, pieces));
            u1 = static_cast<int>(divide(static_cast<int64_t>(tiles) * c1, pieces));
        } else {
            u0 = max(0, c0 - run.fixed);
            u1 = c1 - run.fixed;
            if (u1 <= 0) continue;  // only the fixed cost fell into this run: the next worker has it all
        }
        const int h = task % a.heads, rt = task / a.heads;
        const int row_end = s.rows * a.group;

        // Tokens that every row of the tile sees: no mask inside.
        const int tok_lo = rt * ROWS / a.group, tok_hi = min(s.rows - 1, (rt * ROWS + ROWS - 1) / a.group);
        const int all1 = a.causal ? s.len - s.rows + tok_lo + 1 : s.len;
        const int64_t all0 = a.window > 0 ? static_cast<int64_t>(s.len) - s.rows + tok_hi + 1 - a.window : 0;

        const int32_t* table = a.table + static_cast<int64_t>(b) * a.table_pages;
        const int last = min(u1, seen_tiles);
        const int page_mask = (1 << a.page_shift) - 1;
        const auto page_of = [&](int tile) {
            return tile < last ? table[(see.lo + 16 * tile) >> a.page_shift] : 0;
        };
        // Tiles u0 + warp, u0 + warp + kWarps, ...: the first tiles' page indices,
        // then the query rows, are on their way while addresses are computed.
        const int tile0 = u0 + warp;
        int pages[STAGES];
        #pragma unroll
        for (int i = 0; i < STAGES; ++i) pages[i] = page_of(tile0 + i * kWarps);
        Query<T, DP> q[NT];
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = rt * ROWS + 8 * n + g;
            const int tok = r / a.group, hd = r - tok * a.group;
            const T* row = static_cast<const T*>(a.q) + (s.row0 + tok) * a.q_tok +
                           static_cast<int64_t>(h * a.group + hd) * a.q_head;
            load_query<T, DP>(q[n], row, r < row_end, dim, a.q_vec != 0, t);
        }
        const auto checked = [&](int page, bool& ok) {
            ok = page >= 0 && page < a.pages;
            return ok ? page : 0;
        };
        // The ring: row r's piece c lies at c ^ 4 (r & 1) for keys, of which
        // eight lanes read two rows' half, and at c ^ 2 (r / 2 % 4) for values, of
        // which they read a quarter of rows 0, 2, 4, 6: both without conflicts.
        // (At dim 64 keys need no swizzle and values keep two-way conflicts.)
        const uint32_t ring = smem_ring + worker * R::kRing + warp * STAGES * R::kTileBytes;
        const uint32_t scales = smem_ring + R::kScales + (worker * kWarps + warp) * STAGES * 8;
        const int crow = lane / CH, cpiece = lane % CH;  // of this lane's first copy
        const auto k_place = [&](int r, int c) { return DP == 64 ? c : c ^ (r & 1) << 2; };
        const auto v_place = [&](int r, int c) { return DP == 64 ? c ^ (r >> 1 & 1) << 1 : c ^ (r >> 1 & 3) << 1; };
        unsigned int valid = 0;  // bit s: the page of the tile in stage s is one
        const auto copy = [&](int tile, int stage, int page) {
            bool in;
            page = checked(page, in);
            valid = (valid & ~(1u << stage)) | static_cast<unsigned int>(in) << stage;
            const int64_t at = static_cast<int64_t>(page) * a.heads + h;
            const int64_t off = ((at << a.page_shift) + ((see.lo + 16 * tile) & page_mask)) * dim;
            const uint32_t dst = ring + stage * R::kTileBytes;
            #pragma unroll
            for (int n = 0; n < COPIES; ++n) {
                const int r = crow + n * (32 / CH);
                const int64_t src = off + (FULL ? 16 * lane + 512 * n : r * dim + 16 * cpiece);
                const int bytes = FULL || 16 * cpiece < dim ? 16 : 0;
                cp_async16(dst + r * DP + 16 * k_place(r, cpiece), a.k + (bytes ? src : off), bytes);
                cp_async16(dst + 16 * DP + r * DP + 16 * v_place(r, cpiece), a.v + (bytes ? src : off), bytes);
            }
            if (lane < 2) cp_async4(scales + 8 * stage + 4 * lane, (lane == 0 ? a.ks : a.vs) + at);
        };
        #pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) {
            if (tile0 + i * kWarps < last) copy(tile0 + i * kWarps, i, pages[i]);
            cp_async_commit();
        }
        int page_ahead = pages[STAGES - 1];
        // --- query rows ------------------------------------------------------
        uint32_t qd[NT][DIGITS][DP / 16];
        float fac[NT][2];
        int see0[NT][2], see1[NT][2];  // visible tokens of rows 2 t, 2 t + 1
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float f = query_digits<T, DP, DIGITS>(qd[n], q[n]) * a.scale_log2;
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                fac[n][c] = __shfl_sync(0xffffffffu, f, 4 * (2 * t + c));
                const int rc = rt * ROWS + 8 * n + 2 * t + c;
                const int64_t pos = static_cast<int64_t>(s.len) - s.rows + rc / a.group;
                see1[n][c] = a.causal ? static_cast<int>(max(pos + 1, int64_t{0})) : s.len;
                see0[n][c] = a.window > 0 ? static_cast<int>(max(pos + 1 - a.window, int64_t{0})) : 0;
            }
        }
        float o[NT][NJ][4] = {};
        float m[NT][2], l[NT][2];
        #pragma unroll
        for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.0f;

        int stage = 0;
        for (int tile = tile0; tile < last; tile += kWarps) {
            cp_async_wait_group<STAGES - 2>();
            __syncwarp();
            {
                const int ahead = tile + (STAGES - 1) * kWarps;
                if (ahead < last) copy(ahead, stage == 0 ? STAGES - 1 : stage - 1, page_ahead);
                cp_async_commit();
                page_ahead = page_of(ahead + kWarps);
            }
            const bool ok_now = valid >> stage & 1u;
            const uint32_t at = ring + stage * R::kTileBytes;
            uint32_t kr[2][KP][4];
            #pragma unroll
            for (int r = 0; r < 2; ++r) {
                #pragma unroll
                for (int c = 0; c < KP; ++c) load_shared(kr[r][c], at + (g + 8 * r) * DP + 16 * k_place(g, t + 4 * c));
            }
            uint32_t sv[2];
            load_shared(sv, scales + 8 * stage);
            const float ks_now = nan_unless_finite(__uint_as_float(sv[0])), vs = __uint_as_float(sv[1]);

            int sc[NT][DIGITS][4];
            #pragma unroll
            for (int step = 0; step < DP / 32; ++step) {
                // Words of the step's two halves: pieces 2 i and 2 i + 1, or two
                // words of the only piece.
                constexpr bool ONE = DP == 64;
                const int p0 = ONE ? 0 : 2 * (step / 4), p1 = ONE ? 0 : p0 + 1;
                const int w0 = ONE ? step : step % 4, w1 = ONE ? step + 2 : w0;
                const uint32_t ka[4] = {kr[0][p0][w0], kr[1][p0][w0], kr[0][p1][w1], kr[1][p1][w1]};
                #pragma unroll
                for (int n = 0; n < NT; ++n) {
                    #pragma unroll
                    for (int i = 0; i < DIGITS; ++i) {
                        const uint32_t b0 = qd[n][i][4 * p0 + w0], b1 = qd[n][i][4 * p1 + w1];
                        if (step == 0) mma_s8_16832_from(sc[n][i], ka, b0, b1, kMagicBits);
                        else mma_s8_16832(sc[n][i], ka, b0, b1);
                    }
                }
            }
            // vs = 2^ve vf with vf in [1, 2); scales below 2^-80 belong to
            // all-zero codes, for non-finite ones vf is NaN.
            const uint32_t vbits = __float_as_uint(vs);
            int ve = static_cast<int>((vbits >> 23) & 0xffu) - 127;
            float vf = __uint_as_float((vbits & 0x807fffffu) | 0x3f800000u);
            if (ve == 128) ve = 0, vf = __int_as_float(0x7fffffff);
            if (ve < -80) ve = -80, vf = 0.0f;
            if (!ok_now) ve = 0, vf = 0.0f;
            const float vexp = static_cast<float>(ve), vinv = __int_as_float((127 - ve) << 23);

            const int tok = see.lo + 16 * tile;
            const bool whole = ok_now && tok >= all0 && tok + 16 <= all1;
            float p[NT][4];
            bool grow = false;
            #pragma unroll
            for (int n = 0; n < NT; ++n) {
                #pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float x = __int_as_float(sc[n][DIGITS - 1][c]) - kMagic;
                    #pragma unroll
                    for (int i = DIGITS - 2; i >= 0; --i) {
                        x = fmaf(x, 256.0f, __int_as_float(sc[n][i][c]) - kMagic);
                    }
                    p[n][c] = fmaf(x, fac[n][c & 1] * ks_now, vexp);
                }
                if (!whole) {
                    #pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int j = tok + g + 8 * (c >> 1);
                        if (!ok_now || j < see0[n][c & 1] || j >= see1[n][c & 1] || j >= s.len) p[n][c] = -INFINITY;
                    }
                }
                #pragma unroll
                for (int c = 0; c < 4; ++c) grow = grow || p[n][c] > m[n][c & 1] + kSlack;
            }
            if (__any_sync(0xffffffffu, grow)) {
                #pragma unroll
                for (int n = 0; n < NT; ++n) {
                    #pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float top = fmaxf(p[n][c], p[n][c + 2]);
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        top = fmaxf(top, m[n][c]);
                        const float by = join_factor(m[n][c], top);
                        m[n][c] = top;
                        l[n][c] *= by;
                        #pragma unroll
                        for (int j = 0; j < NJ; ++j) o[n][j][c] *= by, o[n][j][c + 2] *= by;
                    }
                }
            }
            uint32_t hi[NT][2], lo[NT][2];
            #pragma unroll
            for (int n = 0; n < NT; ++n) {
                float e[4];
                #pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float base = m[n][c & 1] == -INFINITY ? 0.0f : m[n][c & 1];
                    const float x = exp2_fast(p[n][c] + (kLift - base));
                    l[n][c & 1] = fmaf(x, vinv, l[n][c & 1]);
                    e[c] = x * vf;
                    if (!whole && p[n][c] == -INFINITY) e[c] = 0.0f;  // hidden from this row: vf may be NaN
                }
                #pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint32_t top = pack_f16(e[2 * r], e[2 * r + 1]);
                    hi[n][r] = transpose8(top);
                    if (SPLIT) {
                        const __half2 th = *reinterpret_cast<const __half2*>(&top);
                        lo[n][r] = transpose8(pack_f16(e[2 * r] - __low2float(th), e[2 * r + 1] - __high2float(th)));
                    }
                }
            }
            uint32_t vr[4][VP][VW];
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 2 * t + (i & 1) + 8 * (i >> 1);
                #pragma unroll
                for (int c = 0; c < VP; ++c) {
                    const uint32_t row = at + 16 * DP + r * DP;
                    if constexpr (DP == 64) load_shared(vr[i][c], row + 16 * v_place(r, g >> 1) + 8 * (g & 1));
                    else load_shared(vr[i][c], row + 16 * v_place(r, g + 8 * c));
                }
            }
            #pragma unroll
            for (int c = 0; c < VP; ++c) {
                #pragma unroll
                for (int w = 0; w < VW; ++w) {
                    // Bytes 0, 1 and 2, 3 of this word, of the token pairs
                    // (2 t, 2 t + 1) and (2 t + 8, 2 t + 9).
                    const uint32_t bias = 0x80808080u;
                    const uint32_t x0 = __byte_perm(vr[0][c][w], vr[1][c][w], 0x5140) ^ bias;
                    const uint32_t y0 = __byte_perm(vr[0][c][w], vr[1][c][w], 0x7362) ^ bias;
                    const uint32_t x1 = __byte_perm(vr[2][c][w], vr[3][c][w], 0x5140) ^ bias;
                    const uint32_t y1 = __byte_perm(vr[2][c][w], vr[3][c][w], 0x7362) ^ bias;
                    const uint32_t va[2][4] = {
                        {codes_f16<0x4140>(x0), codes_f16<0x4342>(x0), codes_f16<0x4140>(x1), codes_f16<0x4342>(x1)},
                        {codes_f16<0x4140>(y0), codes_f16<0x4342>(y0), codes_f16<0x4140>(y1), codes_f16<0x4342>(y1)}};
                    #pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int j = 2 * (VW * c + w) + i;
                        #pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if (FRESH) {
                                float d[4];
                                mma_f16_16816_from(d, va[i], lo[n][0], lo[n][1], 0.0f);
                                mma_f16_16816(d, va[i], hi[n][0], hi[n][1]);
                                #pragma unroll
                                for (int c4 = 0; c4 < 4; ++c4) o[n][j][c4] += d[c4];
                            } else {
                                if (SPLIT) mma_f16_16816(o[n][j], va[i], lo[n][0], lo[n][1]);
                                mma_f16_16816(o[n][j], va[i], hi[n][0], hi[n][1]);
                            }
                        }
                    }
                }
            }
            if (!ok_now && lane == 0) atomicOr(&g_attn_err, kKvErrAttention);
            stage = stage == STAGES - 1 ? 0 : stage + 1;
        }
        cp_async_wait_group<0>();

        // --- join the warps --------------------------------------------------
        sync_worker();  // all tiles have been read
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x = l[n][c];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                const int r = 8 * n + 2 * t + c;
                if (g == 0) s_ml[warp][r][0] = m[n][c], s_ml[warp][r][1] = x;
                // Elements 2 j, 2 j + 1 of the lane's run of dim.
                #pragma unroll
                for (int j = 0; j < NJ; j += 2) {
                    const int run = DP == 64 ? 8 * g : 16 * (g + 8 * (j / 8));
                    *reinterpret_cast<float4*>(&s_o[warp][r][run + 2 * (j % 8)]) =
                        make_float4(o[n][j][c], o[n][j][c + 2], o[n][j + 1][c], o[n][j + 1][c + 2]);
                }
            }
        }
        sync_worker();
        const bool complete = u0 == 0 && u1 == tiles;
        const int64_t slot = 2 * static_cast<int64_t>(run.worker) + (u0 > 0 ? 0 : 1);
        for (int i = tid; i < ROWS * (DP / 4); i += kThreads) {
            const int r = i / (DP / 4), d = 4 * (i % (DP / 4));
            const int row = rt * ROWS + r;
            if (row >= row_end) continue;
            float top = -INFINITY, den = 0.0f, sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            #pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_ml[w][r][0]);
            #pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = join_factor(s_ml[w][r][0], top);
                const float4 x = *reinterpret_cast<const float4*>(&s_o[w][r][d]);
                den = fmaf(s_ml[w][r][1], f, den);
                sum[0] = fmaf(x.x, f, sum[0]), sum[1] = fmaf(x.y, f, sum[1]);
                sum[2] = fmaf(x.z, f, sum[2]), sum[3] = fmaf(x.w, f, sum[3]);
            }
            if (complete) {
                const int tk = row / a.group;
                store_row<T>(a, s.row0 + tk, h * a.group + row - tk * a.group, d, sum, den, top, d == 0);
            } else {
                if (d == 0) a.ml[slot * ROWS + r] = make_float2(top, den);
                *reinterpret_cast<float4*>(a.part + (slot * ROWS + r) * DP + d) =
                    make_float4(sum[0], sum[1], sum[2], sum[3]);
            }
        }
        if (tid == 0 && u0 == 0 && (a.by_task || !complete)) {
            const int more = complete ? 0 : run.piece ? pieces - 1
                                          : owner_of_last(run, from + static_cast<int64_t>(task + 1) * each) - run.worker;
            put_entry(a, run, task0 + task, more, s, task);
        }
        sync_worker();  // the ring is free again
    }
}

// Joins the partial results of one row of one task: block c's second slot,
// then the first slots of the blocks after it, in that order. Four warps take
// every fourth partial. Bound by latency: the entry, then maxima and the first
// four sums of each warp at once, then the output.
template <typename T, int DP, int ROWS>
__global__ void __launch_bounds__(kThreads) kv_join_kernel(const AttnArgs a) {
    constexpr int PER = DP >= 128 ? DP / 128 : 1;  // float4 pieces of a sum per lane
    constexpr int AHEAD = 4;
    __shared__ float s_top[kWarps], s_den[kWarps];
    __shared__ __align__(16) float s_o[kWarps][DP];
    pdl_launch_dependents();
    pdl_wait();
    const int entries = a.entry[0].x;
    const int4 e = a.entry[1 + 2 * blockIdx.x];
    const int task = a.entry[2 + 2 * blockIdx.x].x;
    if (static_cast<int>(blockIdx.x) >= entries || e.x == 0) return;
    const int r = blockIdx.y, h = task % a.heads, row = task / a.heads * ROWS + r;
    if (row >= e.w * a.group) return;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int count = e.x + 1;
    const auto slot = [&](int i) { return static_cast<int64_t>(2 * (e.y + i) + (i == 0 ? 1 : 0)) * ROWS + r; };
    const auto load = [&](int i, float2& ml, float4 (&x)[PER]) {
        ml = a.ml[slot(i)];
        #pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int d = 4 * (lane + 32 * k);
            if (d < DP) x[k] = *reinterpret_cast<const float4*>(a.part + slot(i) * DP + d);
        }
    };
    float2 ml[AHEAD];
    float4 x[AHEAD][PER] = {};
    #pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
        ml[j] = make_float2(-INFINITY, 0.0f);
        if (warp + j * kWarps < count) load(warp + j * kWarps, ml[j], x[j]);
    }
    float top = -INFINITY;
    for (int i = tid; i < count; i += kThreads) top = fmaxf(top, a.ml[slot(i)].x);
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) s_top[warp] = top;
    __syncthreads();
    #pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_top[w]);

    float den = 0.0f, sum[PER][4] = {};
    const auto add = [&](const float2& m, const float4 (&v)[PER]) {
        const float f = join_factor(m.x, top);
        den = fmaf(m.y, f, den);
        #pragma unroll
        for (int k = 0; k < PER; ++k) {
            sum[k][0] = fmaf(v[k].x, f, sum[k][0]), sum[k][1] = fmaf(v[k].y, f, sum[k][1]);
            sum[k][2] = fmaf(v[k].z, f, sum[k][2]), sum[k][3] = fmaf(v[k].w, f, sum[k][3]);
        }
    };
    #pragma unroll
    for (int j = 0; j < AHEAD; ++j) add(ml[j], x[j]);
    #pragma unroll 4
    for (int i = warp + AHEAD * kWarps; i < count; i += kWarps) {
        load(i, ml[0], x[0]);
        add(ml[0], x[0]);
    }
    if (lane == 0) s_den[warp] = den;
    #pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int d = 4 * (lane + 32 * k);
        if (d < DP) *reinterpret_cast<float4*>(&s_o[warp][d]) = make_float4(sum[k][0], sum[k][1], sum[k][2], sum[k][3]);
    }
    __syncthreads();
    const int d = 4 * tid;
    if (d >= DP) return;
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    den = 0.0f;
    #pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        den += s_den[w];
        #pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += s_o[w][d + j];
    }
    const int tk = row / a.group;
    store_row<T>(a, e.z + tk, h * a.group + row - tk * a.group, d, o, den, top, d == 0);
}

// Sets the kernels' shared memory once a device.
template <typename T, int DP, int NT, bool FULL>
cudaError_t rows_ready() {
    constexpr int kDevices = 64;
    static bool ready[kDevices] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < kDevices && __atomic_load_n(&ready[dev], __ATOMIC_RELAXED))) return e;
    e = cudaFuncSetAttribute(kv_rows_kernel<T, DP, NT, FULL>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Rows<T, DP, NT>::kBytes);
    if (e == cudaSuccess && dev < kDevices) __atomic_store_n(&ready[dev], true, __ATOMIC_RELAXED);
    return e;
}

// Launches with the caller's workspace, or only says how many bytes it takes
// (ws_bytes != nullptr).
template <typename T, int DP, int NT, bool FULL>
cudaError_t run_rows(AttnArgs a, int64_t tasks, void* ws, int64_t* ws_bytes, cudaStream_t stream) {
    constexpr int ROWS = 8 * NT;
    const int64_t blocks = device_sm_count(), grid = blocks * Rows<T, DP, NT>::kWorkers;
    const int64_t entry_bytes = (1 + 2 * grid) * sizeof(int4);
    const int64_t ml_bytes = 2 * grid * ROWS * sizeof(float2);
    if (ws_bytes != nullptr) {
        *ws_bytes = entry_bytes + ml_bytes + 2 * grid * ROWS * DP * sizeof(float);
        return cudaSuccess;
    }
    a.by_task = tasks <= grid ? 1 : 0;
    a.entries = static_cast<int>(a.by_task ? tasks : grid);
    a.entry = static_cast<int4*>(ws);
    a.ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + entry_bytes);
    a.part = reinterpret_cast<float*>(static_cast<char*>(ws) + entry_bytes + ml_bytes);
    cudaError_t e = rows_ready<T, DP, NT, FULL>();
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = pdl_config(dim3(static_cast<unsigned>(blocks)), dim3(kThreads * Rows<T, DP, NT>::kWorkers),
                                        Rows<T, DP, NT>::kBytes, stream, attr);
    e = cudaLaunchKernelEx(&cfg, kv_rows_kernel<T, DP, NT, FULL>, a);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3(static_cast<unsigned>(a.entries), ROWS);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, kv_join_kernel<T, DP, ROWS>, a);
}

template <typename T>
cudaError_t run_attention(const AttnArgs& a, int64_t max_tokens, void* ws, int64_t* ws_bytes, cudaStream_t stream) {
    // Tasks of at most 8 or 16 query rows; an upper bound of their number. Two
    // sides of 8 read the codes once for 16 rows and pay where they come from HBM:
    // 64 sequences of 4000 tokens, 8 key heads of 128, 16 rows, bf16: 154 us against
    // 171 with one side, 16 sequences with 32 rows 76 against 82. With less work one
    // side is the faster: 16 sequences with 16 rows 48 against 52, one of 1000 tokens
    // 10.5 against 13.2.
    const bool two = !Traits<T>::kFresh && a.dim <= 128 && max_tokens * a.group > 8;
    const int rows = two ? 16 : 8;
    const int64_t tasks = a.heads * (static_cast<int64_t>(a.tokens) * a.group / rows + a.seqs);
    const auto run = [&](auto dp, auto nt) {
        constexpr int DP = decltype(dp)::value, NT = decltype(nt)::value;
        return a.dim == DP ? run_rows<T, DP, NT, true>(a, tasks, ws, ws_bytes, stream)
                           : run_rows<T, DP, NT, false>(a, tasks, ws, ws_bytes, stream);
    };
    const std::integral_constant<int, 1> one;
    if constexpr (!Traits<T>::kFresh) {
        const std::integral_constant<int, 2> pair;
        if (two && a.dim <= 64) return run(std::integral_constant<int, 64>{}, pair);
        if (two) return run(std::integral_constant<int, 128>{}, pair);
    }
    if (a.dim <= 64) return run(std::integral_constant<int, 64>{}, one);
    if (a.dim <= 128) return run(std::integral_constant<int, 128>{}, one);
    return run(std::integral_constant<int, 256>{}, one);
}

cudaError_t run_rows_typed(popcornType_t type, const AttnArgs& a, int64_t max_tokens, void* ws, int64_t* ws_bytes,
                           cudaStream_t stream) {
    switch (type) {
        case POPCORN_TYPE_F32: return run_attention<float>(a, max_tokens, ws, ws_bytes, stream);
        case POPCORN_TYPE_F16: return run_attention<__half>(a, max_tokens, ws, ws_bytes, stream);
        default: return run_attention<__nv_bfloat16>(a, max_tokens, ws, ws_bytes, stream);
    }
}

// Launches the kernel, or the two, that the sizes ask for; with ws_bytes only
// says how much workspace they take, for any block table if a.table_pages is 0.
// Sequences of less than kPromptRows query rows go to kv_rows_kernel and others
// to the prompt kernel, each of which skips the other's; where tokens are seqs
// times max_tokens only the prompt kernel is launched, and in small calls only
// kv_rows_kernel. One that is alone takes sequences of any number of rows: `first`,
// which only the device knows, may end before `tokens` and leave some with fewer.
cudaError_t run_typed(popcornType_t type, AttnArgs a, int64_t max_tokens, void* ws, int64_t* ws_bytes,
                      cudaStream_t stream) {
    a.min_rows = 1, a.max_rows = INT32_MAX;
    max_tokens = std::min(max_tokens, static_cast<int64_t>(a.tokens));
    const int64_t tasks = a.heads * (static_cast<int64_t>(a.tokens) * a.group / 16 + a.seqs);
    const bool small = tasks <= device_sm_count() && tasks * (a.table_pages << a.page_shift) <= kFewTokens;
    if (max_tokens * a.group < kPromptRows || !prompt_supported(type, a.dim) || (small && a.table_pages > 0)) {
        return run_rows_typed(type, a, max_tokens, ws, ws_bytes, stream);
    }
    const bool both = a.tokens != max_tokens * a.seqs;
    const int64_t few = (kPromptRows - 1) / a.group;  // queries of a sequence that kv_rows_kernel keeps
    AttnArgs rows = a;
    rows.max_rows = kPromptRows - 1;
    if (both) a.min_rows = kPromptRows;
    cudaError_t e = cudaSuccess;
    if (ws_bytes != nullptr) {
        int64_t prompt = 0, beside = 0, alone = 0;
        e = run_prompt(type, a, nullptr, &prompt, stream);
        if (e == cudaSuccess && both && few > 0) e = run_rows_typed(type, rows, few, nullptr, &beside, stream);
        if (e == cudaSuccess && small) e = run_rows_typed(type, rows, max_tokens, nullptr, &alone, stream);
        *ws_bytes = std::max({prompt, beside, alone});
        return e;
    }
    e = run_prompt(type, a, ws, nullptr, stream);
    if (e == cudaSuccess && both && few > 0) e = run_rows_typed(type, rows, few, ws, nullptr, stream);
    return e;
}

// Argument checks that the workspace query shares with the call.
bool attention_supported(const popcornKvCache_t& c, popcornType_t type, int64_t seqs, int64_t tokens,
                         int64_t max_tokens, int64_t q_heads) {
    return kv_cache_supported(c) && kv_type_supported(type) && q_heads > 0 && q_heads <= 65535 &&
           q_heads % c.heads == 0 && max_tokens > 0 && seqs <= INT32_MAX / 2 && tokens <= INT32_MAX / q_heads;
}

AttnArgs attention_sizes(const popcornKvCache_t& c, int64_t seqs, int64_t tokens, int64_t q_heads) {
    AttnArgs a = {};
    a.pages = c.pages;
    a.seqs = static_cast<int>(seqs), a.tokens = static_cast<int>(tokens);
    a.heads = static_cast<int>(c.heads), a.group = static_cast<int>(q_heads / c.heads);
    a.dim = static_cast<int>(c.dim), a.page_shift = log2_of(c.page_size);
    return a;
}

}  // namespace

cudaError_t kv_attention_take_errors(unsigned int* bits) {
    const unsigned int zero = 0;
    unsigned int prompt = 0;
    cudaError_t e = cudaMemcpyFromSymbol(bits, g_attn_err, sizeof(unsigned int));
    if (e == cudaSuccess && *bits != 0) e = cudaMemcpyToSymbol(g_attn_err, &zero, sizeof(unsigned int));
    if (e == cudaSuccess) e = kv_prompt_take_errors(&prompt);
    *bits |= prompt;
    return e;
}

}  // namespace pcb

extern "C" int64_t popcornKvAttentionWorkspace(const popcornKvCache_t* cache, popcornType_t type, int64_t seqs,
                                               int64_t tokens, int64_t max_tokens, int64_t q_heads) {
    if (cache == nullptr || seqs <= 0 || tokens <= 0 ||
        !pcb::attention_supported(*cache, type, seqs, tokens, max_tokens, q_heads)) {
        return 0;
    }
    int64_t bytes = 0;
    const pcb::AttnArgs a = pcb::attention_sizes(*cache, seqs, tokens, q_heads);
    const cudaError_t e = pcb::run_typed(type, a, max_tokens, nullptr, &bytes, nullptr);
    return pcb::record_cuda(e) == POPCORN_SUCCESS ? bytes : 0;
}

extern "C" popcornStatus_t popcornKvAttention(void* out, float* lse, const void* q, int64_t q_token_stride,
                                              int64_t q_head_stride, popcornType_t type, const popcornKvCache_t* cache,
                                              const int32_t* table, int64_t table_pages, const int32_t* first,
                                              const int32_t* length, int64_t seqs, int64_t tokens, int64_t max_tokens,
                                              int64_t q_heads, int causal, int64_t window, float scale,
                                              void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
    if (out == nullptr || q == nullptr || cache == nullptr || cache->k == nullptr || cache->v == nullptr ||
        cache->k_scale == nullptr || cache->v_scale == nullptr || table == nullptr || length == nullptr) {
        return POPCORN_ERROR_INVALID_VALUE;
    }
    if (seqs <= 0 || tokens <= 0) return POPCORN_SUCCESS;
    // Positions and row counts are 32-bit inside a sequence; the kernel for
    // prompts counts up to 255 tokens past the last one.
    if (!pcb::attention_supported(*cache, type, seqs, tokens, max_tokens, q_heads) || table_pages <= 0 ||
        table_pages > (INT32_MAX - 256) / cache->page_size || !pcb::aligned16(out) ||
        (first == nullptr && tokens != seqs)) {
        return POPCORN_ERROR_INVALID_VALUE;
    }
    pcb::AttnArgs a = pcb::attention_sizes(*cache, seqs, tokens, q_heads);
    a.out = out, a.lse = lse, a.q = q, a.q_tok = q_token_stride, a.q_head = q_head_stride;
    a.k = cache->k, a.v = cache->v, a.ks = cache->k_scale, a.vs = cache->v_scale;
    a.table = table, a.first = first, a.length = length;
    // (Positions are below 2^31: a window of that many tokens hides none.)
    a.table_pages = table_pages, a.window = window > INT32_MAX ? 0 : window, a.causal = causal;
    a.scale_log2 = scale * 1.4426950408889634f;
    const int64_t four = 4 * pcb::kv_type_size(type);
    a.q_vec = reinterpret_cast<uintptr_t>(q) % four == 0 && q_token_stride % 4 == 0 && q_head_stride % 4 == 0;

    // A caller's workspace has the size that the query gives, for any block table.
    int64_t need = 0;
    pcb::AttnArgs sizes = a;
    if (workspace != nullptr) sizes.table_pages = 0;
    cudaError_t e = pcb::run_typed(type, sizes, max_tokens, nullptr, &need, stream);
    if (e != cudaSuccess) return pcb::record_cuda(e);
    void* ws = workspace;
    if (workspace == nullptr) {
        e = pcb::scratch_alloc(&ws, static_cast<size_t>(need), stream);
        if (e != cudaSuccess) return pcb::record_cuda(e);
    } else if (workspace_bytes < need || !pcb::aligned16(workspace)) {
        return POPCORN_ERROR_INVALID_VALUE;
    }
    e = pcb::run_typed(type, a, max_tokens, ws, nullptr, stream);
    if (workspace == nullptr) {
        const cudaError_t f = pcb::scratch_free(ws, stream);
        if (e == cudaSuccess) e = f;
    }
    if (e != cudaSuccess) return pcb::record_cuda(e);
    return pcb::check_launch();
}
