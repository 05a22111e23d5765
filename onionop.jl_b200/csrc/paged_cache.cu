// Writing a paged key-value cache and cutting it back (addressing: paged.cuh).
//
// Append: the new tokens' K and V rows into their pages, K (and the queries)
// rotated by RoPE on the way where cos/sin are given -- the rotation, the copy of V
// and the scatter in one launch.  Bound: HBM, each byte read and written once.
//
// Evict: per (sequence, KV head) the `budget` slots to keep -- the last `recent`
// ones and the heaviest of the others by accumulated attention weight -- and their
// rows moved, in order, to the pages of another table.  Bound: HBM, 4 bytes per
// slot for the choice and 4·E·size bytes per kept slot for the move.
#include "paged.cuh"

namespace nnop {
namespace paged {

int check_cache(const char* who, Cache& c, const int32_t* table, const int32_t* lengths, int64_t E, int64_t KH,
                int64_t B, int64_t pages, int64_t page_size, int64_t max_pages, int64_t page_stride,
                int64_t head_stride, int64_t row_stride, int dtype) {
    const std::string w(who);
    if (dtype != NNOP_F32 && dtype != NNOP_F16 && dtype != NNOP_BF16)
        return fail(NNOP_ERR_DTYPE, w + ": unsupported dtype " + std::to_string(dtype));
    if (E <= 0 || KH <= 0 || B < 0 || pages < 0 || page_size <= 0 || max_pages < 0)
        return fail(NNOP_ERR_SHAPE, w + ": invalid dimensions");
    if ((E & (E - 1)) != 0) return fail(NNOP_ERR_SHAPE, "Only power-of-2 embedding dims are supported.");
    if (E < 16 || E > 128)
        return fail(NNOP_ERR_SHAPE, w + ": embedding dim " + std::to_string(E) + " not supported (16, 32, 64, 128)");
    if (KH > 65535 || B > 65535) return fail(NNOP_ERR_SHAPE, w + ": too many heads or sequences");
    const int64_t most = ((int64_t)1 << 31) - 1024;
    if (pages > most || page_size > most || max_pages > most || page_size * max_pages > most)
        return fail(NNOP_ERR_SHAPE, w + ": more than 2^31 - 1024 pages or slots per sequence");
    const int64_t vec = dtype == NNOP_F32 ? 4 : 8;
    if (page_stride < 0 || head_stride < 0 || row_stride < 0)
        return fail(NNOP_ERR_SHAPE, w + ": negative cache stride");
    if (page_stride % vec || head_stride % vec || row_stride % vec)
        return fail(NNOP_ERR_ALIGN, w + ": cache strides must be multiples of 16 bytes");
    if (B > 0 && (!lengths || (max_pages > 0 && !table))) return fail(NNOP_ERR_ARG, w + ": NULL pointer");
    c.table = table;
    c.lengths = lengths;
    c.pages = pages;
    c.max_pages = max_pages;
    c.page_stride = page_stride;
    c.head_stride = head_stride;
    c.row_stride = row_stride;
    c.slots = (int)(page_size * max_pages);
    c.page_size = FastDiv((uint32_t)page_size);
    return NNOP_OK;
}

namespace {

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
struct AppendArgs {
    const void *q, *k, *v;
    const float *cos_t, *sin_t;
    const int* n_new;
    void *q_out, *k_cache, *v_cache;
    int* new_lengths;
    Cache c;
    int64_t T, B, cos_batch;
    int QH, KH;
};

constexpr int kAppendBlock = 256;

// A thread owns one 16-byte vector of the first half of a (head, token) row and its
// partner E/2 further on: the pair that RoPE rotates.
template <typename T, int E>
__global__ void __launch_bounds__(kAppendBlock) append_kernel(AppendArgs a) {
    constexpr int VEC = 16 / sizeof(T), HALF = E / 2, NH = HALF / VEC;
    const int heads = a.QH + 2 * a.KH;      // rows of q, then k, then v
    const int64_t total = a.B * heads * a.T * NH;
    const int64_t first = (int64_t)blockIdx.x * kAppendBlock + threadIdx.x;
    if (first < a.B) {
        const int n = a.n_new ? min(max(a.n_new[first], 0), (int)a.T) : (int)a.T;
        a.new_lengths[first] = (int)min((int64_t)a.c.length(first) + n, (int64_t)a.c.slots);
    }
    for (int64_t i = first; i < total; i += (int64_t)gridDim.x * kAppendBlock) {
        const int u = (int)(i % NH);
        int64_t r = i / NH;
        const int t = (int)(r % a.T);
        r /= a.T;
        const int h = (int)(r % heads);
        const int64_t b = r / heads;
        const bool is_q = h < a.QH, is_v = h >= a.QH + a.KH;
        const T* src;
        T* dst;
        if (is_q) {
            const int64_t off = ((b * a.QH + h) * a.T + t) * E;
            src = static_cast<const T*>(a.q) + off;
            dst = static_cast<T*>(a.q_out) + off;
        } else {
            const int n = a.n_new ? min(a.n_new[b], (int)a.T) : (int)a.T;
            const int64_t slot = (int64_t)a.c.length(b) + t;
            if (t >= n || slot >= a.c.slots) continue;
            const int kvh = h - a.QH - (is_v ? a.KH : 0);
            const int64_t to = a.c.offset(a.c.table + b * a.c.max_pages, (int)slot, (int64_t)kvh * a.c.head_stride);
            if (to < 0) continue;
            src = static_cast<const T*>(is_v ? a.v : a.k) + ((b * a.KH + kvh) * a.T + t) * E;
            dst = static_cast<T*>(is_v ? a.v_cache : a.k_cache) + to;
        }
        Vec<T, VEC> x = ldg_stream<T, VEC>(src + u * VEC), y = ldg_stream<T, VEC>(src + u * VEC + HALF);
        if (!is_v && a.cos_t != nullptr) {
            const int64_t at = ((a.cos_batch == 1 ? 0 : b) * a.T + t) * E + u * VEC;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float c = __ldg(a.cos_t + at + e), s = __ldg(a.sin_t + at + e);
                // the order of roundings that nnop_llama_rope's results have
                const float x1 = to_f(x.v[e]), x2 = to_f(y.v[e]);
                x.v[e] = from_f<T>(fmaf(x1, c, -__fmul_rn(x2, s)));
                y.v[e] = from_f<T>(fmaf(x2, c, __fmul_rn(x1, s)));
            }
        }
        *reinterpret_cast<Vec<T, VEC>*>(dst + u * VEC) = x;
        *reinterpret_cast<Vec<T, VEC>*>(dst + u * VEC + HALF) = y;
    }
}

template <typename T, int E>
int launch_append(const AppendArgs& a, cudaStream_t s) {
    constexpr int NH = E / 2 / (16 / (int)sizeof(T));
    const int64_t items = std::max(a.B * (a.QH + 2 * a.KH) * a.T * NH, a.B);
    const int64_t grid = std::min((items + kAppendBlock - 1) / kAppendBlock, (int64_t)1 << 30);
    append_kernel<T, E><<<(unsigned)grid, kAppendBlock, 0, s>>>(a);
    return check_launch("paged_append");
}

// ---------------------------------------------------------------------------
// evict
// ---------------------------------------------------------------------------
struct EvictArgs {
    const float* weights;
    int* new_lengths;
    float* new_weights;      // [B][KH][new_slots]
    int* kept;               // [B][KH][budget]
    const int* new_table;    // [B][new_max_pages]
    void *k_cache, *v_cache;
    Cache c;
    int64_t B, new_max_pages;
    int KH, budget, recent, new_slots;
};

// Order-preserving key of a weight: a larger weight has the larger key, −0 equals +0,
// NaN is above every number.
__device__ __forceinline__ uint32_t order_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

constexpr int kSelectThreads = 1024;

// One CTA per (sequence, KV head): the (budget − recent)-th largest weight by four
// counting passes over 8 bits each, then the kept slots in order.
__global__ void __launch_bounds__(kSelectThreads) evict_select(EvictArgs a) {
    __shared__ int hist[256];
    __shared__ int pick[2];
    __shared__ int warp_gt[32], warp_eq[32];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int64_t b = blockIdx.x / a.KH;
    const float* w = a.weights + (int64_t)blockIdx.x * a.c.slots;
    float* nw = a.new_weights + (int64_t)blockIdx.x * a.new_slots;
    int* kept = a.kept + (int64_t)blockIdx.x * a.budget;
    const int n = a.c.length(b), count = min(n, a.budget);
    if (blockIdx.x % a.KH == 0 && t == 0) a.new_lengths[b] = count;
    for (int i = count + t; i < a.budget; i += kSelectThreads) kept[i] = -1;
    for (int i = count + t; i < a.new_slots; i += kSelectThreads) nw[i] = 0.f;
    const int last = n <= a.budget ? n : min(a.recent, a.budget);   // slots kept unseen
    const int cand = n - last;
    const int need = count - last;                                  // of the first `cand`
    for (int i = t; i < last; i += kSelectThreads) {
        kept[need + i] = cand + i;
        nw[need + i] = w[cand + i];
    }
    if (need == 0) return;
    uint32_t prefix = 0;
    int rank = need;            // the wanted key is the rank-th largest of those with this prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (t < 256) hist[t] = 0;
        __syncthreads();
        for (int i = t; i < cand; i += kSelectThreads) {
            const uint32_t key = order_key(w[i]);
            if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
        }
        __syncthreads();
        if (t == 0) {
            int d = 255, r = rank;
            while (hist[d] < r) r -= hist[d--];
            pick[0] = d;
            pick[1] = r;
        }
        __syncthreads();
        prefix = prefix << 8 | (uint32_t)pick[0];
        rank = pick[1];
    }
    // keys above `prefix` are kept, and the first `rank` that equal it
    int gt = 0, eq = 0;         // in front of this tile
    for (int i0 = 0; i0 < cand; i0 += kSelectThreads) {
        const int i = i0 + t;
        const float x = i < cand ? w[i] : 0.f;
        const uint32_t key = order_key(x);
        const bool is_gt = i < cand && key > prefix, is_eq = i < cand && key == prefix;
        const uint32_t mg = __ballot_sync(0xffffffffu, is_gt), me = __ballot_sync(0xffffffffu, is_eq);
        if (lane == 0) {
            warp_gt[warp] = __popc(mg);
            warp_eq[warp] = __popc(me);
        }
        __syncthreads();
        int g = gt + __popc(mg & ((1u << lane) - 1)), e = eq + __popc(me & ((1u << lane) - 1));
        for (int k = 0; k < 32; ++k) {
            if (k < warp) {
                g += warp_gt[k];
                e += warp_eq[k];
            }
            gt += warp_gt[k];
            eq += warp_eq[k];
        }
        if (is_gt || (is_eq && e < rank)) {
            const int at = g + min(e, rank);
            kept[at] = i;
            nw[at] = x;
        }
        __syncthreads();
    }
}

constexpr int kMoveBlock = 256;

// Moves the kept rows: a thread moves one 16-byte vector of K or V.
template <typename T, int E>
__global__ void __launch_bounds__(kMoveBlock) evict_move(EvictArgs a) {
    constexpr int VEC = 16 / sizeof(T), NV = E / VEC;
    wait_before();
    const int64_t total = a.B * a.KH * a.budget * (2 * NV);
    for (int64_t i = (int64_t)blockIdx.x * kMoveBlock + threadIdx.x; i < total; i += (int64_t)gridDim.x * kMoveBlock) {
        const int u = (int)(i % (2 * NV));
        int64_t r = i / (2 * NV);
        const int at = (int)(r % a.budget);
        r /= a.budget;
        const int h = (int)(r % a.KH);
        const int64_t b = r / a.KH;
        const int slot = a.kept[r * a.budget + at];
        if (slot < 0) continue;
        const int64_t ho = (int64_t)h * a.c.head_stride;
        const int64_t from = a.c.offset(a.c.table + b * a.c.max_pages, slot, ho);
        const int64_t to = a.c.offset(a.new_table + b * a.new_max_pages, at, ho);
        if (from < 0 || to < 0) continue;
        T* pool = static_cast<T*>(u < NV ? a.k_cache : a.v_cache);
        const int e = (u < NV ? u : u - NV) * VEC;
        *reinterpret_cast<Vec<T, VEC>*>(pool + to + e) = *reinterpret_cast<const Vec<T, VEC>*>(pool + from + e);
    }
}

template <typename T, int E>
int launch_evict(const EvictArgs& a, cudaStream_t s) {
    constexpr int NV = E / (16 / (int)sizeof(T));
    evict_select<<<(unsigned)(a.B * a.KH), kSelectThreads, 0, s>>>(a);
    if (const int rc = check_launch("paged_evict")) return rc;
    const int64_t items = a.B * a.KH * a.budget * 2 * NV;
    if (items == 0) return NNOP_OK;
    const int64_t grid = std::min((items + kMoveBlock - 1) / kMoveBlock, (int64_t)1 << 30);
    return launch_dependent("paged_evict", evict_move<T, E>, dim3((unsigned)grid), dim3(kMoveBlock), 0, s, a);
}

}  // namespace
}  // namespace paged
}  // namespace nnop

using namespace nnop;

#define NNOP_DISPATCH_E(E, EC, ...)                         \
    switch (E) {                                            \
        case 16: { constexpr int EC = 16; __VA_ARGS__; }    \
        case 32: { constexpr int EC = 32; __VA_ARGS__; }    \
        case 64: { constexpr int EC = 64; __VA_ARGS__; }    \
        default: { constexpr int EC = 128; __VA_ARGS__; }   \
    }

extern "C" {

int nnop_paged_append(const void* q, const void* k, const void* v, const float* cos_t, const float* sin_t,
                      const int32_t* n_new, void* q_out, void* k_cache, void* v_cache, const int32_t* block_table,
                      const int32_t* lengths, int32_t* new_lengths, int64_t E, int64_t T, int64_t QH, int64_t KH,
                      int64_t B, int64_t cos_batch, int64_t pages, int64_t page_size, int64_t max_pages,
                      int64_t page_stride, int64_t head_stride, int64_t row_stride, int dtype, void* stream) {
    return paged::guarded("paged_append", [&]() -> int {
        paged::AppendArgs a{};
        if (const int rc = paged::check_cache("paged_append", a.c, block_table, lengths, E, KH, B, pages, page_size,
                                              max_pages, page_stride, head_stride, row_stride, dtype))
            return rc;
        if (T < 0 || QH < 0 || QH > 65535 || T > ((int64_t)1 << 31) - 1024)
            return fail(NNOP_ERR_SHAPE, "paged_append: invalid dimensions");
        if ((cos_t != nullptr) != (sin_t != nullptr) || (QH == 0 && q) ||
            (QH > 0 && T > 0 && B > 0 && (!q || !q_out || !cos_t)))
            return fail(NNOP_ERR_ARG, "paged_append: cos and sin come together, and q (QH > 0) with them");
        if (cos_t && cos_batch != B && cos_batch != 1)
            return fail(NNOP_ERR_SHAPE, "paged_append: cos/sin batch must equal the batch or be 1");
        if (B == 0) return NNOP_OK;
        if (!new_lengths || new_lengths == lengths || (T > 0 && (!k || !v)) || (pages > 0 && (!k_cache || !v_cache)))
            return fail(NNOP_ERR_ARG, "paged_append: NULL pointer, or new_lengths is lengths");
        if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_out) || !aligned16(k_cache) || !aligned16(v_cache))
            return fail(NNOP_ERR_ALIGN, "paged_append: tensors must be 16-byte aligned");
        a.q = q;
        a.k = k;
        a.v = v;
        a.cos_t = cos_t;
        a.sin_t = sin_t;
        a.n_new = n_new;
        a.q_out = q_out;
        a.k_cache = k_cache;
        a.v_cache = v_cache;
        a.new_lengths = new_lengths;
        a.T = T;
        a.B = B;
        a.cos_batch = cos_batch;
        a.QH = (int)QH;
        a.KH = (int)KH;
        const cudaStream_t s = (cudaStream_t)stream;
        NNOP_DISPATCH_DTYPE(dtype, D, { NNOP_DISPATCH_E(E, EC, return paged::launch_append<D, EC>(a, s)) });
        return NNOP_OK;
    });
}

int nnop_paged_evict(void* k_cache, void* v_cache, const int32_t* block_table, const int32_t* new_table,
                     const int32_t* lengths, const float* weights, int32_t* new_lengths, float* new_weights,
                     int32_t* kept, int64_t E, int64_t KH, int64_t B, int64_t pages, int64_t page_size,
                     int64_t max_pages, int64_t new_max_pages, int64_t page_stride, int64_t head_stride,
                     int64_t row_stride, int64_t budget, int64_t recent, int dtype, void* stream) {
    return paged::guarded("paged_evict", [&]() -> int {
        paged::EvictArgs a{};
        if (const int rc = paged::check_cache("paged_evict", a.c, block_table, lengths, E, KH, B, pages, page_size,
                                              max_pages, page_stride, head_stride, row_stride, dtype))
            return rc;
        const int64_t most = ((int64_t)1 << 31) - 1024;
        if (new_max_pages < 0 || new_max_pages > most || new_max_pages * page_size > most)
            return fail(NNOP_ERR_SHAPE, "paged_evict: more than 2^31 - 1024 slots per sequence");
        if (budget < 0 || recent < 0 || recent > budget || budget > new_max_pages * page_size)
            return fail(NNOP_ERR_SHAPE, "paged_evict: 0 <= recent <= budget <= slots of the new table");
        if (B == 0) return NNOP_OK;
        if (!new_lengths || new_lengths == lengths || (a.c.slots > 0 && !weights) ||
            (new_max_pages > 0 && (!new_weights || !new_table)) || (budget > 0 && !kept) ||
            (pages > 0 && (!k_cache || !v_cache)))
            return fail(NNOP_ERR_ARG, "paged_evict: NULL pointer, or new_lengths is lengths");
        if (new_weights != nullptr && new_weights == weights)
            return fail(NNOP_ERR_ARG, "paged_evict: new_weights is weights");
        if (!aligned16(k_cache) || !aligned16(v_cache))
            return fail(NNOP_ERR_ALIGN, "paged_evict: tensors must be 16-byte aligned");
        if (B * KH > most) return fail(NNOP_ERR_SHAPE, "paged_evict: too many heads or sequences");
        a.weights = weights;
        a.new_lengths = new_lengths;
        a.new_weights = new_weights;
        a.kept = kept;
        a.new_table = new_table;
        a.k_cache = k_cache;
        a.v_cache = v_cache;
        a.B = B;
        a.new_max_pages = new_max_pages;
        a.KH = (int)KH;
        a.budget = (int)budget;
        a.recent = (int)recent;
        a.new_slots = (int)(new_max_pages * page_size);
        const cudaStream_t s = (cudaStream_t)stream;
        NNOP_DISPATCH_DTYPE(dtype, D, { NNOP_DISPATCH_E(E, EC, return paged::launch_evict<D, EC>(a, s)) });
        return NNOP_OK;
    });
}

}  // extern "C"
