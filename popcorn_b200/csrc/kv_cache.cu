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
// bandwidth; at prompts it streams.
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

// Elements 4 i .. 4 i + 3 of a row, rotated (rot > 0) by the row's cos / sin.
// Products and sums are rounded one by one so that a restatement in separate
// f32 operations gives the same bits.
template <typename T>
__device__ __forceinline__ void rotated4(const T* row, int i, int rot, bool interleaved, const float* cos,
                                         const float* sin, bool vec, float (&v)[4]) {
    const int d = 4 * i;
    load4(row + d, vec, v);
    if (d >= rot) return;
    const int half = rot >> 1;
    if (interleaved) {
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float c = cos[2 * i + j], s = sin[2 * i + j];
            const float a = v[2 * j], b = v[2 * j + 1];
            v[2 * j] = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
            v[2 * j + 1] = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
        }
        return;
    }
    const bool low = d < half;
    const int k = low ? d : d - half;
    float p[4], c[4], s[4];
    load4(row + (low ? d + half : d - half), vec, p);
    load4(cos + k, vec, c);
    load4(sin + k, vec, s);
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float own = __fmul_rn(v[j], c[j]), other = __fmul_rn(p[j], s[j]);
        v[j] = low ? __fsub_rn(own, other) : __fadd_rn(own, other);
    }
}

__device__ __forceinline__ int encode(float x, float s) {
    // rint of the quotient, clamped; NaN (0 / 0, inf / inf) becomes 0.
    return s > 0.0f ? max(-128, min(127, __float2int_rn(__fdiv_rn(x, s)))) : 0;
}

// THREADS threads per block: the first half works on keys, the second on
// values. CQ: 4-element groups of the new rows that a thread keeps in
// registers between the maximum and the encoding; what does not fit is read
// (from L1 or L2) and rotated again. Decode (few new rows a block) runs one
// warp for each half, prompts four.
template <typename T, int THREADS, int CQ>
__global__ void __launch_bounds__(THREADS) append_kernel(const AppendArgs a) {
    constexpr int H = THREADS / 2;
    __shared__ float part[THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31;
    const bool vec = a.vec != 0;
    const int quads = a.dim >> 2;

    if (blockIdx.x >= a.blocks) {  // queries: one token's heads, split over q_parts blocks
        const int64_t qb = blockIdx.x - a.blocks;
        const int64_t t = qb / a.q_parts;
        const int64_t b = a.first ? sequence_of(a.first, a.seqs, t, lane) : t;
        if (b >= a.seqs) return;
        const int64_t pos = a.start[b] + (a.first ? t - a.first[b] : 0);
        if (a.rot > 0 && (pos < 0 || pos >= a.positions)) {
            if (tid == 0) atomicOr(&g_kv_err, kKvErrAppend);
            return;
        }
        const float* cos = a.cos + pos * (a.rot >> 1);
        const float* sin = a.sin + pos * (a.rot >> 1);
        const int total = a.q_heads * quads;
        const T* q = static_cast<const T*>(a.q) + t * a.q_tok;
        T* o = static_cast<T*>(a.q_out) + t * a.q_heads * a.dim;
        // A rotated pair's two halves may lie in different threads, and q_out
        // may be q: each batch of heads is read whole, then written.
        const int part_i = static_cast<int>(qb % a.q_parts);
        const int heads_each = (a.q_heads + a.q_parts - 1) / a.q_parts;
        const int lo = part_i * heads_each * quads, hi = min(total, lo + heads_each * quads);
        const int step = max(1, (THREADS * 4) / quads) * quads;  // whole heads
        for (int base = lo; base < hi; base += step) {
            const int end = min(hi, base + step);
            float v[4][4];
            #pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = base + tid + u * THREADS;
                if (i < end) {
                    const int h = i / quads;
                    rotated4(q + h * a.q_head, i - h * quads, a.rot, a.interleaved != 0, cos, sin, vec, v[u]);
                }
            }
            __syncthreads();
            #pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = base + tid + u * THREADS;
                if (i < end) store4(o + 4 * i, a.q_vec != 0, v[u]);
            }
        }
        return;
    }

    const int kv = tid / H, ht = tid % H;
    const int64_t slot = blockIdx.x / a.heads;
    const int h = static_cast<int>(blockIdx.x % a.heads);
    const int64_t t_end = min(a.tokens, (slot + 1) * a.chunk);
    const T* x = static_cast<const T*>(a.x[kv]) + h * a.head[kv];
    const int rot = kv == 0 ? a.rot : 0;
    const int page_size = 1 << a.page_shift;

    for (int64_t t = slot * a.chunk; t < t_end;) {
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
        const int total = n * quads;

        float v[CQ][4];
        float m = 0.0f;
        #pragma unroll
        for (int u = 0; u < CQ; ++u) {
            const int i = ht + u * H;
            if (i < total) {
                const int r = i / quads;
                rotated4(x + (t + r) * a.tok[kv], i - r * quads, rot, a.interleaved != 0,
                         a.cos + (pos + r) * (a.rot >> 1), a.sin + (pos + r) * (a.rot >> 1), vec, v[u]);
                #pragma unroll
                for (int j = 0; j < 4; ++j) m = fmaxf(m, fabsf(v[u][j]));
            }
        }
        for (int i = ht + CQ * H; i < total; i += H) {
            const int r = i / quads;
            float w[4];
            rotated4(x + (t + r) * a.tok[kv], i - r * quads, rot, a.interleaved != 0,
                     a.cos + (pos + r) * (a.rot >> 1), a.sin + (pos + r) * (a.rot >> 1), vec, w);
            #pragma unroll
            for (int j = 0; j < 4; ++j) m = fmaxf(m, fabsf(w[j]));
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
                    uint32_t r = 0;
                    #pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float f = static_cast<float>(static_cast<int8_t>(e[j] >> (8 * k)));
                        r |= (static_cast<uint32_t>(__float2int_rn(__fmul_rn(f, ratio))) & 0xffu) << (8 * k);
                    }
                    e[j] = r;
                }
                w[i] = c;
            }
        }
        uint32_t* w = reinterpret_cast<uint32_t*>(codes + row * a.dim);
        #pragma unroll
        for (int u = 0; u < CQ; ++u) {
            const int i = ht + u * H;
            if (i < total) {
                uint32_t r = 0;
                #pragma unroll
                for (int j = 0; j < 4; ++j) r |= (static_cast<uint32_t>(encode(v[u][j], s)) & 0xffu) << (8 * j);
                w[i] = r;
            }
        }
        for (int i = ht + CQ * H; i < total; i += H) {
            const int r = i / quads;
            float f[4];
            rotated4(x + (t + r) * a.tok[kv], i - r * quads, rot, a.interleaved != 0,
                     a.cos + (pos + r) * (a.rot >> 1), a.sin + (pos + r) * (a.rot >> 1), vec, f);
            uint32_t c = 0;
            #pragma unroll
            for (int j = 0; j < 4; ++j) c |= (static_cast<uint32_t>(encode(f[j], s)) & 0xffu) << (8 * j);
            w[i] = c;
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
    return few ? cudaLaunchKernelEx(&cfg, append_kernel<T, 64, 4>, a)
               : cudaLaunchKernelEx(&cfg, append_kernel<T, 256, 16>, a);
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

    // A slot covers as many tokens as a sequence brings on average, up to a
    // page: at decode every token is its own slot, so that blocks of different
    // sequences run side by side; at prompts a slot holds about one block.
    const int64_t each = tokens / seqs;
    a.chunk = static_cast<int>(each < 1 ? 1 : each > cache->page_size ? cache->page_size : each);
    const bool few = each < 8;
    a.blocks = pcb::ceil_div(tokens, a.chunk) * cache->heads;
    const int threads = few ? 64 : 256;
    a.q_parts = static_cast<int>(q != nullptr ? pcb::ceil_div(q_heads * (cache->dim / 4), threads * 4) : 1);

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
