// Paged 8-bit key/value cache: append (with the position rotation of keys and
// queries) and read-back.
//
// Append. The unit of work is one (page, head) block that gets new rows: its
// scale is shared by all its rows, so one group of threads has to see the
// block's new rows whole. With s the block's old scale (0 where the call
// begins the page) and a = max|new| over the block's new rows,
//   s' = max(s, a / 127),  old code c -> rint(c (s / s')) if s' > s,
//   new value x -> rint(x / s').
// Bytes that it cannot do without: the new rows (read), their codes and the
// scales (written), and the block's earlier codes only where the scale grew.
// At decode that is a few KB a block, so the call is bound by launch and the
// chain first/start -> table -> scale -> codes (four dependent loads), not by
// bandwidth. At prompts instructions count as much as HBM. Measured in a graph,
// append and read-back of the touched pages (in brackets: each alone): a token for
// one sequence 4.7 us (3.0 and 1.8), a token for each of 64 7.9 us (3.9 and 4.3, the
// read-back at 4.8 TB/s), 4 ragged prompts of up to 2048 tokens in f32 with 32 query
// heads rotated 67 us (54 and 8.8, 5.6 TB/s). Tried there and no faster: two query
// tokens a block, blocks of queries and of keys taking turns, more units held in
// registers (72), more blocks an SM. 16-bit prompts take as long as f32 ones (4 up
// to 2048 tokens in bf16: 68 us), although they move half as much.
#include "kv.cuh"

namespace pcb {
namespace {

__device__ unsigned int g_kv_err = 0;

struct AppendArgs {
    int8_t* codes[2];   // keys, values
    float* scale[2];
    const void* x[2];
    int64_t tok[2], head[2];  // strides in elements
    const int32_t* table;
    const int32_t* first;
    const int32_t* start;
    const float* cos;
    const float* sin;
    const void* q;
    void* q_out;
    int64_t q_tok, q_head;
    int64_t pages, table_pages, seqs, tokens, positions;
    int heads, dim, page_shift, rot, interleaved, q_heads;
    int vec;             // every row and table starts on a four-element boundary
    int q_vec;           // so does q_out
    int chunk;           // tokens per slot
    int64_t blocks;      // grid blocks that append; the rest rotate queries
    int q_parts;         // blocks per query token
};

// A row of dim elements in units that rotate by themselves: with the halves
// paired, unit u < rot / 8 is the two groups of four 4 u and 4 u + rot / 2,
// the units after it are single groups; with neighbours paired (or without
// rotation) every unit is a single group. Element index of a unit's first
// group, and whether it has a second one (at + rot / 2).
struct Unit {
    int at;
    bool pair;
};
__device__ __forceinline__ Unit unit_of(int u, int rot, bool interleaved) {
    if (interleaved || u >= (rot >> 3)) return {4 * (interleaved ? u : u + (rot >> 3)), false};
    return {4 * u, true};
}

// A unit's elements, rotated by the row's cos / sin. Products and sums are
// rounded one by one so that a restatement in separate f32 operations gives
// the same bits.
template <typename T>
__device__ __forceinline__ void load_unit(const T* row, Unit u, int rot, bool vec, float (&v)[8]) {
    float lo[4], hi[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    load4(row + u.at, vec, lo);
    if (u.pair) load4(row + u.at + (rot >> 1), vec, hi);
    #pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = lo[j], v[4 + j] = hi[j];
}
__device__ __forceinline__ void turn_unit(Unit u, int rot, const float* cos, const float* sin, bool vec,
                                          float (&v)[8]) {
    if (u.pair) {
        float c[4], s[4];
        load4(cos + u.at, vec, c);
        load4(sin + u.at, vec, s);
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float a = v[j], b = v[4 + j];
            v[j] = __fsub_rn(__fmul_rn(a, c[j]), __fmul_rn(b, s[j]));
            v[4 + j] = __fadd_rn(__fmul_rn(b, c[j]), __fmul_rn(a, s[j]));
        }
    } else if (u.at < rot) {  // neighbours paired
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float c = cos[(u.at >> 1) + j], s = sin[(u.at >> 1) + j];
            const float a = v[2 * j], b = v[2 * j + 1];
            v[2 * j] = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
            v[2 * j + 1] = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
        }
    }
}

__device__ __forceinline__ int encode(float x, float s) {
    // rint of the quotient, clamped; NaN (0 / 0, inf / inf) becomes 0.
    return s > 0.0f ? max(-128, min(127, __float2int_rn(__fdiv_rn(x, s)))) : 0;
}
// rint of a value up to 2^22 in magnitude: the low bits of the sum and the sum
// less the constant (1.5 2^23).
constexpr float kRound = 12582912.0f;
__device__ __forceinline__ uint32_t low_bytes(const float (&t)[4]) {
    const uint32_t a = __byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040);
    const uint32_t b = __byte_perm(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040);
    return __byte_perm(a, b, 0x5410);
}
// Four codes. FAST: v * by, with by = 1 / s, is within 1e-4 of v / s (|v| <=
// 127 s), so that its rint is the quotient's unless it lies near a half; only
// then, and for NaN, there are divisions. At prompts that took 3 us off the 69 of
// the prompts above; at decode a thread has one or two values and the reciprocal
// stands before them (8.2 us against 7.9).
template <bool FAST>
__device__ __forceinline__ uint32_t encode4(const float* v, float s, float by) {
    if (!FAST) {
        uint32_t r = 0;
        #pragma unroll
        for (int j = 0; j < 4; ++j) r |= (static_cast<uint32_t>(encode(v[j], s)) & 0xffu) << (8 * j);
        return r;
    }
    float t[4];
    bool clear = s > 0.0f;
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float y = __fmul_rn(v[j], by);
        t[j] = __fadd_rn(y, kRound);
        clear = clear && fabsf(y - __fsub_rn(t[j], kRound)) <= 0.4999f;
    }
    if (clear) return low_bytes(t);
    uint32_t r = 0;
    #pragma unroll 1
    for (int j = 0; j < 4; ++j) r |= (static_cast<uint32_t>(encode(v[j], s)) & 0xffu) << (8 * j);
    return r;
}

// THREADS threads per block: the first half works on keys, the second on
// values. CU: units of the new rows that a thread keeps in registers between
// the maximum and the encoding; what does not fit is read (from L1 or L2) and
// rotated again. Decode (few new rows a block) runs one warp for each half,
// prompts four.
template <typename T, int THREADS, int CU>
__global__ void __launch_bounds__(THREADS, THREADS == 64 ? 12 : 4) append_kernel(const AppendArgs a) {
    constexpr int H = THREADS / 2;
    constexpr bool FAST = THREADS > 64;
    __shared__ float part[THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31;
    const bool vec = a.vec != 0, inter = a.interleaved != 0;
    const int q_units = a.dim / 4 - (inter ? 0 : a.rot >> 3);

    if (blockIdx.x >= a.blocks) {  // queries: one token's heads, split over q_parts blocks
        const int64_t qb = blockIdx.x - a.blocks;
        const int64_t t = qb / a.q_parts;
        const int part_i = static_cast<int>(qb % a.q_parts);
        const int total = a.q_heads * q_units;
        const T* q = static_cast<const T*>(a.q) + t * a.q_tok;
        T* o = static_cast<T*>(a.q_out) + t * a.q_heads * a.dim;
        float v[2][8];
        #pragma unroll
        for (int u = 0; u < 2; ++u) {  // the rows first: their loads need no position
            const int i = (part_i * 2 + u) * THREADS + tid, h = i / q_units;
            if (i < total) load_unit(q + h * a.q_head, unit_of(i - h * q_units, a.rot, inter), a.rot, vec, v[u]);
        }
        const int64_t b = a.first ? sequence_of(a.first, a.seqs, t, lane) : t;
        const int64_t in = a.first ? t - a.first[b] : 0;
        if (b >= a.seqs || in < 0) return;  // a row of no sequence
        const int64_t pos = a.start[b] + in;
        if (a.rot > 0 && (pos < 0 || pos >= a.positions)) {
            if (tid == 0) atomicOr(&g_kv_err, kKvErrAppend);
            return;
        }
        #pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = (part_i * 2 + u) * THREADS + tid, h = i / q_units;
            if (i >= total) break;
            const Unit un = unit_of(i - h * q_units, a.rot, inter);
            turn_unit(un, a.rot, a.cos + pos * (a.rot >> 1), a.sin + pos * (a.rot >> 1), vec, v[u]);
            const float lo[4] = {v[u][0], v[u][1], v[u][2], v[u][3]}, hi[4] = {v[u][4], v[u][5], v[u][6], v[u][7]};
            store4(o + h * a.dim + un.at, a.q_vec != 0, lo);
            if (un.pair) store4(o + h * a.dim + un.at + (a.rot >> 1), a.q_vec != 0, hi);
        }
        return;
    }

    const int kv = tid / H, ht = tid % H;
    const int64_t slot = blockIdx.x / a.heads;
    const int h = static_cast<int>(blockIdx.x % a.heads);
    const int64_t t_end = min(a.tokens, (slot + 1) * a.chunk);
    const T* x = static_cast<const T*>(a.x[kv]) + h * a.head[kv];
    const int rot = kv == 0 ? a.rot : 0;
    const int units = kv == 0 ? q_units : a.dim >> 2;
    const int page_size = 1 << a.page_shift;

    // (Rows before first[0] belong to no sequence.)
    for (int64_t t = a.first ? max(slot * a.chunk, static_cast<int64_t>(a.first[0])) : slot * a.chunk; t < t_end;) {
        const int64_t b = a.first ? sequence_of(a.first, a.seqs, t, lane) : t;
        if (b >= a.seqs) return;
        const int64_t t0 = a.first ? a.first[b] : t, t1 = a.first ? min(a.tokens, static_cast<int64_t>(a.first[b + 1])) : t + 1;
        const int64_t pos = a.start[b] + (t - t0);
        const int row = static_cast<int>(pos & (page_size - 1));
        // (t + 1: a `first` that does not ascend must not stop the walk.)
        const int64_t next = max(t + 1, min(t1, t + (page_size - row)));
        // Rows t .. next - 1 are the block's new ones if t begins the page or
        // the sequence; else an earlier slot holds the first of them and does
        // the work.
        if (t < t0 || (t > t0 && row > 0)) {
            t = next;
            continue;
        }
        const int n = static_cast<int>(next - t);
        const int64_t at = pos >> a.page_shift;
        int64_t page = -1;
        if (pos >= 0 && at < a.table_pages) page = a.table[b * a.table_pages + at];
        if (page < 0 || page >= a.pages || (a.rot > 0 && pos + n > a.positions)) {
            if (tid == 0) atomicOr(&g_kv_err, kKvErrAppend);
            t = next;
            continue;
        }
        const int64_t block = page * a.heads + h;
        int8_t* codes = a.codes[kv] + (block << a.page_shift) * a.dim;
        const float old = row == 0 ? 0.0f : a.scale[kv][block];

        // This thread's units are H apart: unit c of row r, then the next.
        const int dr = H / units, dc = H - dr * units, r_first = ht / units, c_first = ht - r_first * units;
        const auto step = [&](int& r, int& c) {
            r += dr, c += dc;
            if (c >= units) c -= units, ++r;
        };
        const auto rotated = [&](int r, int c, Unit& un, float (&v)[8]) {  // returns the element index in the block
            un = unit_of(c, rot, inter);
            load_unit(x + (t + r) * a.tok[kv], un, rot, vec, v);
            if (rot > 0) turn_unit(un, rot, a.cos + (pos + r) * (rot >> 1), a.sin + (pos + r) * (rot >> 1), vec, v);
            return (row + r) * a.dim + un.at;
        };
        const auto put = [&](int e, Unit un, const float (&v)[8], float s, float by) {
            *reinterpret_cast<uint32_t*>(codes + e) = encode4<FAST>(v, s, by);
            if (un.pair) *reinterpret_cast<uint32_t*>(codes + e + (rot >> 1)) = encode4<FAST>(v + 4, s, by);
        };
        float v[CU][8];
        float m = 0.0f;
        int r = r_first, c = c_first;
        #pragma unroll
        for (int u = 0; u < CU; ++u, step(r, c)) {
            Unit un;
            if (r < n) {
                rotated(r, c, un, v[u]);
                #pragma unroll
                for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[u][j]));  // (a single group's rest is zero)
            }
        }
        for (; r < n; step(r, c)) {
            Unit un;
            float w[8];
            rotated(r, c, un, w);
            #pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(w[j]));
        }
        // |x| as an unsigned integer keeps its order (no NaN: fmaxf dropped them).
        m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
        if (H > 32) {
            __syncthreads();
            if (lane == 0) part[tid >> 5] = m;
            __syncthreads();
            #pragma unroll
            for (int w = 0; w < H / 32; ++w) m = fmaxf(m, part[kv * (H / 32) + w]);
        }
        float now = __fdiv_rn(m, 127.0f);
        if (now < kKvSmallestScale) now = 0.0f;
        const float s = old > now || old != old ? old : now;

        if (row > 0 && s != old) {
            const float ratio = __fdiv_rn(old, s);
            uint4* w = reinterpret_cast<uint4*>(codes);
            for (int i = ht; i < (row * a.dim) >> 4; i += H) {
                uint4 c = w[i];
                uint32_t* e = reinterpret_cast<uint32_t*>(&c);
                #pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float f[4];
                    #pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        f[k] = __fadd_rn(__fmul_rn(static_cast<float>(static_cast<int8_t>(e[j] >> (8 * k))), ratio), kRound);
                    }
                    e[j] = low_bytes(f);
                }
                w[i] = c;
            }
        }
        const float by = FAST ? __fdiv_rn(1.0f, s) : 0.0f;
        r = r_first, c = c_first;
        #pragma unroll
        for (int u = 0; u < CU; ++u, step(r, c)) {
            const Unit un = unit_of(c, rot, inter);
            if (r < n) put((row + r) * a.dim + un.at, un, v[u], s, by);
        }
        for (; r < n; step(r, c)) {
            Unit un;
            float w[8];
            const int e = rotated(r, c, un, w);
            put(e, un, w, s, by);
        }
        __syncwarp();  // every lane has read the old scale
        if (ht == 0 && (row == 0 || s != old)) a.scale[kv][block] = s;
        t = next;
    }
}

// One block per (listed page, head) and keys or values: 16 bytes of output a
// thread and step, the codes of a step one coalesced load. (No read-only
// loads here or above: under programmatic dependent launch the kernel is
// already running while the previous one writes what it reads.)
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(T* k_out, T* v_out, const int8_t* k, const int8_t* v,
                                                   const float* k_scale, const float* v_scale, const int32_t* list,
                                                   int64_t pages, int heads, int block_codes) {
    constexpr int E = 16 / sizeof(T);  // values per 16-byte store
    pdl_launch_dependents();
    pdl_wait();
    const int64_t i = blockIdx.x / heads;
    const int h = static_cast<int>(blockIdx.x % heads);
    const bool val = blockIdx.y != 0;
    const int64_t page = list[i];
    const bool ok = page >= 0 && page < pages;
    if (!ok && threadIdx.x == 0) atomicOr(&g_kv_err, kKvErrAppend);
    const int64_t block = (ok ? page : 0) * heads + h;
    const int8_t* src = (val ? v : k) + block * block_codes;
    const float s = (val ? v_scale : k_scale)[block];
    uint4* dst = reinterpret_cast<uint4*>((val ? v_out : k_out) + static_cast<int64_t>(blockIdx.x) * block_codes);
    #pragma unroll 4
    for (int j = threadIdx.x; j < block_codes / E; j += 256) {
        alignas(8) int8_t c[E];
        if constexpr (E == 4) {
            *reinterpret_cast<uint32_t*>(c) = reinterpret_cast<const uint32_t*>(src)[j];
        } else {
            *reinterpret_cast<uint2*>(c) = reinterpret_cast<const uint2*>(src)[j];
        }
        uint4 o;
        T* e = reinterpret_cast<T*>(&o);
        #pragma unroll
        for (int n = 0; n < E; ++n) e[n] = from_f32<T>(ok ? __fmul_rn(static_cast<float>(c[n]), s) : 0.0f);
        dst[j] = o;
    }
}

template <typename T>
cudaError_t launch_append(const AppendArgs& a, bool few, cudaStream_t stream) {
    const int threads = few ? 64 : 256;
    const int64_t grid = a.blocks + (a.q ? a.tokens * a.q_parts : 0);
    if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = pdl_config(dim3(static_cast<unsigned>(grid)), dim3(threads), 0, stream, attr);
    return few ? cudaLaunchKernelEx(&cfg, append_kernel<T, 64, 2>, a)
               : cudaLaunchKernelEx(&cfg, append_kernel<T, 256, 2>, a);
}

template <typename T>
cudaError_t launch_read(void* k_out, void* v_out, const popcornKvCache_t& c, const int32_t* list, int64_t count,
                        cudaStream_t stream) {
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg =
        pdl_config(dim3(static_cast<unsigned>(count * c.heads), 2), dim3(256), 0, stream, attr);
    return cudaLaunchKernelEx(&cfg, read_kernel<T>, static_cast<T*>(k_out), static_cast<T*>(v_out),
                              static_cast<const int8_t*>(c.k), static_cast<const int8_t*>(c.v),
                              static_cast<const float*>(c.k_scale), static_cast<const float*>(c.v_scale), list,
                              c.pages, static_cast<int>(c.heads), static_cast<int>(c.page_size * c.dim));
}

bool aligned_to(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace

cudaError_t kv_take_errors(unsigned int* bits) {
    const unsigned int zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(bits, g_kv_err, sizeof(unsigned int));
    if (e == cudaSuccess && *bits != 0) e = cudaMemcpyToSymbol(g_kv_err, &zero, sizeof(unsigned int));
    return e;
}

}  // namespace pcb

extern "C" popcornStatus_t popcornKvAppend(const popcornKvCache_t* cache, const void* k, int64_t k_token_stride,
                                           int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                           int64_t v_head_stride, popcornType_t type, const int32_t* table,
                                           int64_t table_pages, const int32_t* first, const int32_t* start,
                                           int64_t seqs, int64_t tokens, void* q_out, const void* q,
                                           int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads,
                                           const float* cos, const float* sin, int64_t positions, int64_t rot_dim,
                                           int interleaved, cudaStream_t stream) {
    if (cache == nullptr || cache->k == nullptr || cache->v == nullptr || cache->k_scale == nullptr ||
        cache->v_scale == nullptr || k == nullptr || v == nullptr || table == nullptr || start == nullptr) {
        return POPCORN_ERROR_INVALID_VALUE;
    }
    if ((q == nullptr) != (q_out == nullptr) || (cos == nullptr) != (sin == nullptr)) {
        return POPCORN_ERROR_INVALID_VALUE;
    }
    if (seqs <= 0 || tokens <= 0) return POPCORN_SUCCESS;
    if (!pcb::kv_cache_supported(*cache) || !pcb::kv_type_supported(type) || table_pages <= 0) {
        return POPCORN_ERROR_INVALID_VALUE;
    }
    if ((first == nullptr && tokens != seqs) || seqs > INT32_MAX || tokens > INT32_MAX) {
        return POPCORN_ERROR_INVALID_VALUE;
    }
    if (q != nullptr && (q_heads <= 0 || q_heads > 65535)) return POPCORN_ERROR_INVALID_VALUE;
    if (cos != nullptr && (rot_dim <= 0 || rot_dim % 8 != 0 || rot_dim > cache->dim || positions <= 0)) {
        return POPCORN_ERROR_INVALID_VALUE;
    }
    // Writing q_out over q is only defined element for element.
    if (q != nullptr && q_out == q && (q_head_stride != cache->dim || q_token_stride != q_heads * cache->dim)) {
        return POPCORN_ERROR_INVALID_VALUE;
    }

    pcb::AppendArgs a = {};
    a.codes[0] = cache->k, a.codes[1] = cache->v;
    a.scale[0] = cache->k_scale, a.scale[1] = cache->v_scale;
    a.x[0] = k, a.x[1] = v;
    a.tok[0] = k_token_stride, a.tok[1] = v_token_stride;
    a.head[0] = k_head_stride, a.head[1] = v_head_stride;
    a.table = table, a.first = first, a.start = start;
    a.rot = cos != nullptr ? static_cast<int>(rot_dim) : 0;
    a.cos = cos, a.sin = sin, a.positions = positions, a.interleaved = interleaved;
    a.q = q, a.q_out = q_out, a.q_tok = q_token_stride, a.q_head = q_head_stride;
    a.q_heads = static_cast<int>(q_heads);
    a.pages = cache->pages, a.table_pages = table_pages, a.seqs = seqs, a.tokens = tokens;
    a.heads = static_cast<int>(cache->heads), a.dim = static_cast<int>(cache->dim);
    a.page_shift = pcb::log2_of(cache->page_size);

    const int64_t four = 4 * pcb::kv_type_size(type);
    bool vec = pcb::aligned_to(k, four) && pcb::aligned_to(v, four) && k_token_stride % 4 == 0 &&
               k_head_stride % 4 == 0 && v_token_stride % 4 == 0 && v_head_stride % 4 == 0;
    if (q != nullptr) vec = vec && pcb::aligned_to(q, four) && q_token_stride % 4 == 0 && q_head_stride % 4 == 0;
    if (cos != nullptr) vec = vec && pcb::aligned16(cos) && pcb::aligned16(sin);
    a.vec = vec ? 1 : 0;
    a.q_vec = pcb::aligned_to(q_out, four) ? 1 : 0;

    // A slot's blocks are worked on one after the other. At prompts (a page of
    // tokens a sequence and more) a slot of a page's length holds about one
    // block; below, slots of a quarter of a sequence's tokens keep blocks of
    // different sequences side by side, at decode each token is its own slot.
    // (Threads of a block, 8 key heads of 128, 64 against 256: 5 tokens for each of
    // 64 sequences in f32 7.4 against 10.3 us, 8 tokens 11.4 against 10.3; 8 tokens
    // for each of 16 in bf16 8.2 against 4.8, 4 tokens 5.2 against 4.2.)
    const int64_t each = tokens / seqs;
    a.chunk = static_cast<int>(each >= cache->page_size ? cache->page_size : each < 8 ? 1 : each / 4);
    const bool few = each < 8;
    a.blocks = pcb::ceil_div(tokens, a.chunk) * cache->heads;
    const int threads = few ? 64 : 256;
    const int64_t units = cache->dim / 4 - (interleaved ? 0 : a.rot / 8);
    a.q_parts = static_cast<int>(q != nullptr ? pcb::ceil_div(q_heads * units, threads * 2) : 1);

    cudaError_t e;
    switch (type) {
        case POPCORN_TYPE_F32: e = pcb::launch_append<float>(a, few, stream); break;
        case POPCORN_TYPE_F16: e = pcb::launch_append<__half>(a, few, stream); break;
        default: e = pcb::launch_append<__nv_bfloat16>(a, few, stream); break;
    }
    if (e != cudaSuccess) return pcb::record_cuda(e);
    return pcb::check_launch();
}

extern "C" popcornStatus_t popcornKvRead(void* k_out, void* v_out, popcornType_t type, const popcornKvCache_t* cache,
                                         const int32_t* list, int64_t count, cudaStream_t stream) {
    if (cache == nullptr || cache->k == nullptr || cache->v == nullptr || cache->k_scale == nullptr ||
        cache->v_scale == nullptr || k_out == nullptr || v_out == nullptr || list == nullptr) {
        return POPCORN_ERROR_INVALID_VALUE;
    }
    if (count <= 0) return POPCORN_SUCCESS;
    if (!pcb::kv_cache_supported(*cache) || !pcb::kv_type_supported(type) || !pcb::aligned16(k_out) ||
        !pcb::aligned16(v_out) || count > INT32_MAX / cache->heads) {
        return POPCORN_ERROR_INVALID_VALUE;
    }
    cudaError_t e;
    switch (type) {
        case POPCORN_TYPE_F32: e = pcb::launch_read<float>(k_out, v_out, *cache, list, count, stream); break;
        case POPCORN_TYPE_F16: e = pcb::launch_read<__half>(k_out, v_out, *cache, list, count, stream); break;
        default: e = pcb::launch_read<__nv_bfloat16>(k_out, v_out, *cache, list, count, stream); break;
    }
    if (e != cudaSuccess) return pcb::record_cuda(e);
    return pcb::check_launch();
}
