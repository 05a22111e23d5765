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

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

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
    c.pages = (uint32_t)pages;
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
    FastDiv T;
    int64_t tokens, B, cos_batch;      // tokens = B·T
    int QH, KH;
};

constexpr int kAppendBlock = 256;
constexpr int kAppendHeads = 4;      // heads per thread

// A thread owns one 16-byte vector of the first half of a token's rows and its partner
// E/2 further on (the pair that RoPE rotates) for kAppendHeads heads of q, of k or of v
// (blockIdx.y): the angles, the page and the index arithmetic are fetched once for all
// of them, and all rows are loaded before any is used.  Four prompts of 8192 tokens (32 +
// 8 heads of 128, bf16, 772 MB), the launch alone: 117 us, 6.59 TB/s, with streaming stores
// (a call through the Python mirror: 121 us, 6.4 TB/s); 175 us with plain ones, 126 with
// two heads per thread, 117 with eight.
template <typename T, int E>
__global__ void __launch_bounds__(kAppendBlock) append_kernel(AppendArgs a) {
    constexpr int VEC = 16 / sizeof(T), HALF = E / 2, NH = HALF / VEC;
    const int64_t i = (int64_t)blockIdx.x * kAppendBlock + threadIdx.x;
    if (blockIdx.y == 0 && i < a.B) {
        const int most = a.tokens > 0 ? (int)a.T.d : 0;
        const int n = a.n_new ? min(max(a.n_new[i], 0), most) : most;
        a.new_lengths[i] = (int)min((int64_t)a.c.length(i) + n, (int64_t)a.c.slots);
    }
    if (i >= a.tokens * NH) return;
    const int u = (int)(i % NH);
    const uint32_t r = (uint32_t)(i / NH);
    const int64_t b = a.T.div(r);
    const int t = (int)(r - (uint32_t)b * a.T.d);
    const int gq = (a.QH + kAppendHeads - 1) / kAppendHeads, gk = (a.KH + kAppendHeads - 1) / kAppendHeads;
    const int g = blockIdx.y;
    const bool is_q = g < gq, is_v = g >= gq + gk;
    const int h0 = (is_q ? g : is_v ? g - gq - gk : g - gq) * kAppendHeads;
    const int H = is_q ? a.QH : a.KH;
    const int64_t step = (int64_t)a.T.d * E;       // between heads of the new rows
    const int64_t at = ((b * H + h0) * a.T.d + t) * E + u * VEC;
    const T* src = static_cast<const T*>(is_q ? a.q : is_v ? a.v : a.k) + at;
    T* dst;
    int64_t dst_step;
    if (is_q) {
        dst = static_cast<T*>(a.q_out) + at;
        dst_step = step;
    } else {
        const int64_t slot = (int64_t)a.c.length(b) + t;
        if ((a.n_new && t >= a.n_new[b]) || slot >= a.c.slots) return;
        const int64_t to = a.c.offset(a.c.table + b * a.c.max_pages, (int)slot);
        if (to < 0) return;
        dst = static_cast<T*>(is_v ? a.v_cache : a.k_cache) + to + h0 * a.c.head_stride + u * VEC;
        dst_step = a.c.head_stride;
    }
    Vec<T, VEC> x[kAppendHeads], y[kAppendHeads];
#pragma unroll
    for (int j = 0; j < kAppendHeads; ++j)
        if (h0 + j < H) {
            x[j] = ldg_stream<T, VEC>(src + j * step);
            y[j] = ldg_stream<T, VEC>(src + j * step + HALF);
        }
    if (!is_v && a.cos_t != nullptr) {
        const int64_t ca = ((a.cos_batch == 1 ? 0 : b) * a.T.d + t) * E + u * VEC;
        float c[VEC], s[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            c[e] = __ldg(a.cos_t + ca + e);
            s[e] = __ldg(a.sin_t + ca + e);
        }
#pragma unroll
        for (int j = 0; j < kAppendHeads; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                // the order of roundings that nnop_llama_rope's results have
                const float x1 = to_f(x[j].v[e]), x2 = to_f(y[j].v[e]);
                x[j].v[e] = from_f<T>(fmaf(x1, c[e], -__fmul_rn(x2, s[e])));
                y[j].v[e] = from_f<T>(fmaf(x2, c[e], __fmul_rn(x1, s[e])));
            }
    }
#pragma unroll
    for (int j = 0; j < kAppendHeads; ++j)
        if (h0 + j < H) {
            st_stream<T, VEC>(dst + j * dst_step, x[j]);
            st_stream<T, VEC>(dst + j * dst_step + HALF, y[j]);
        }
}

template <typename T, int E>
int launch_append(const AppendArgs& a, cudaStream_t s) {
    constexpr int NH = E / 2 / (16 / (int)sizeof(T));
    const int64_t items = std::max(a.tokens * NH, a.B);
    const unsigned grid = (unsigned)((items + kAppendBlock - 1) / kAppendBlock);
    const unsigned groups = (a.QH + kAppendHeads - 1) / kAppendHeads + 2 * ((a.KH + kAppendHeads - 1) / kAppendHeads);
    append_kernel<T, E><<<dim3(grid, groups), kAppendBlock, 0, s>>>(a);
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
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kDigits = 3;                                   // of 11, 11 and 10 bits
constexpr int kBins = 2048;
constexpr size_t kHistBytes = sizeof(int) * kDigits * kBins;
constexpr int kMostKeys = 48 * 1024;                         // of a CTA's share in shared memory

constexpr int kMostCtas = 8;                                 // of a cluster
// The kernel counts slots with 32-bit numbers in steps of up to its whole cluster, and the
// last step goes past the end.
constexpr int64_t kMostEvictSlots = ((int64_t)1 << 31) - kMostCtas * kSelectThreads;
static_assert(kMostCtas * kSelectThreads >= 4 * kSelectThreads, "a thread takes four keys of its CTA's share a step");

// Sum over the lanes in front.
__device__ __forceinline__ int warp_sum_before(int n) {
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if ((threadIdx.x & 31) >= o) incl += up;
    }
    return incl - n;
}

__device__ __forceinline__ int digit_shift(int d) { return d == 0 ? 21 : d == 1 ? 10 : 0; }

// The slots to keep of one (sequence, KV head): a cluster of 1 to 8 CTAs, each with a
// contiguous share of the slots and its keys in shared memory (read once; a share of
// more than kMostKeys is read again).  The (budget − recent)-th largest key is found
// digit by digit: every CTA counts its keys by the digit and gives every CTA of the
// cluster its counts of 32 bins at once; one warp of each finds the 32 bins that the
// wanted key is in, fetches those of the other CTAs through distributed shared memory
// and finds the bin (all 2048 bins of 8 CTAs, fetched by all threads, take 4 us a digit).
// Then each CTA writes its kept slots in order, behind those of the CTAs in front of it: a
// slot's place is (larger keys in front) + min(equal keys in front, equals to keep).
__global__ void __launch_bounds__(kSelectThreads) evict_select(EvictArgs a, int most_keys) {
    extern __shared__ __align__(16) int smem[];
    int* hist = smem;                                        // [kDigits][kBins]
    uint32_t* keys = reinterpret_cast<uint32_t*>(smem + kDigits * kBins);
    __shared__ int pick[2], warp_gt[kSelectWarps], warp_eq[kSelectWarps], mine[2];
    __shared__ __align__(8) int coarse[kDigits][kMostCtas][kBins / 32];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    let_next_start();
    const int64_t row = blockIdx.x / C;
    const int64_t b = row / a.KH;
    const float* w = a.weights + row * a.c.slots;
    float* nw = a.new_weights + row * a.new_slots;
    int* kept = a.kept + row * a.budget;
    const int n = a.c.length(b), count = min(n, a.budget);
    const int gt0 = rank * kSelectThreads + t, all = C * kSelectThreads;
    if (row % a.KH == 0 && gt0 == 0) a.new_lengths[b] = count;
    for (int i = count + gt0; i < a.budget; i += all) kept[i] = -1;
    for (int i = count + gt0; i < a.new_slots; i += all) nw[i] = 0.f;
    const int last = n <= a.budget ? n : min(a.recent, a.budget);   // slots kept unseen
    const int cand = n - last;
    const int need = count - last;                                  // of the first `cand`
    for (int i = gt0; i < last; i += all) kept[need + i] = cand + i;
    if (need == 0) return;                                   // the same for the whole cluster
    auto begun = cluster.barrier_arrive();
    const int share = (cand + C - 1) / C;
    const int i0 = min(rank * share, cand), size = min(share, cand - i0);
    const bool held = size <= most_keys;
    for (int i = t; i < kDigits * kBins; i += kSelectThreads) hist[i] = 0;
    if (held) {
#pragma unroll 8
        for (int i = t; i < size; i += kSelectThreads) keys[i] = order_key(w[i0 + i]);
    }
    cluster.barrier_wait(std::move(begun));      // every CTA runs: its shared memory may be written
    __syncthreads();                             // this one's counts are zero, its keys there
    // Four keys from i (a multiple of 4); 0, which is no number's key, behind the last.
    auto four = [&](int i) {
        uint4 k = make_uint4(0, 0, 0, 0);
        if (held) k = *reinterpret_cast<const uint4*>(keys + i);
        else {
            k.x = order_key(w[i0 + i]);
            if (i + 1 < size) k.y = order_key(w[i0 + i + 1]);
            if (i + 2 < size) k.z = order_key(w[i0 + i + 2]);
            if (i + 3 < size) k.w = order_key(w[i0 + i + 3]);
        }
        if (i + 1 >= size) k.y = 0;
        if (i + 2 >= size) k.z = 0;
        if (i + 3 >= size) k.w = 0;
        return k;
    };
    uint32_t prefix = 0;        // digits of the wanted key so far
    int left = need;            // it is the left-th largest of the keys that begin so
#pragma unroll
    for (int d = 0; d < kDigits; ++d) {
        const int shift = digit_shift(d), above = d == 0 ? 0 : digit_shift(d - 1);
        const int bins = d == 2 ? 1024 : 2048;
        int* h = hist + d * kBins;
        auto add = [&](uint32_t key) {
            if (key != 0 && (d == 0 || key >> above == prefix)) atomicAdd(&h[(key >> shift) & (bins - 1)], 1);
        };
        for (int i = 4 * t; i < size; i += 4 * kSelectThreads) {
            const uint4 k = four(i);
            add(k.x);
            add(k.y);
            add(k.z);
            add(k.w);
        }
        __syncthreads();
        // counts of 32 bins: 16 threads with two bins each; lane c of them writes to CTA c
        if (2 * t < bins) {
            const int2 two = *reinterpret_cast<const int2*>(h + 2 * t);
            const int of32 = __reduce_add_sync(lane < 16 ? 0xffffu : 0xffff0000u, two.x + two.y);
            if ((lane & 15) < C) cluster.map_shared_rank(&coarse[d][rank][t / 16], lane & 15)[0] = of32;
        }
        cluster.sync();
        if (warp == 0) {
            // the wanted key's 32 bins, then its bin: lane l has the l-th from the top
            const int last32 = bins / 32 - 1 - 2 * lane;
            int n1 = 0, n0 = 0;
            if (last32 > 0) {
#pragma unroll
                for (int c = 0; c < kMostCtas; ++c) {
                    if (c >= C) break;
                    const int2 x = *reinterpret_cast<const int2*>(&coarse[d][c][last32 - 1]);
                    n0 += x.x;
                    n1 += x.y;
                }
            }
            int over = warp_sum_before(n0 + n1);
            int in = -1;
            if (over < left && left <= over + n1) in = last32;
            else if (over + n1 < left && left <= over + n1 + n0) {
                in = last32 - 1;
                over += n1;
            }
            const int who = __ffs(__ballot_sync(0xffffffffu, in >= 0)) - 1;
            in = __shfl_sync(0xffffffffu, in, who);
            const int rest = left - __shfl_sync(0xffffffffu, over, who);
            const int bin = in * 32 + 31 - lane;
            int from[kMostCtas];
#pragma unroll
            for (int c = 0; c < kMostCtas; ++c)
                from[c] = c == rank ? h[bin] : c < C ? cluster.map_shared_rank(h, c)[bin] : 0;
            int sum = 0;
#pragma unroll
            for (int c = 0; c < kMostCtas; ++c) sum += from[c];
            over = warp_sum_before(sum);
            if (over < rest && rest <= over + sum) {
                pick[0] = bin;
                pick[1] = rest - over;
            }
        }
        __syncthreads();
        prefix = prefix << (d == 2 ? 10 : 11) | (uint32_t)pick[0];
        left = pick[1];
    }
    // Larger keys are kept, and the first `left` that equal it.  Each warp has a contiguous
    // run, each lane four slots of 128.
    const int run = ((size + kSelectWarps - 1) / kSelectWarps + 127) & ~127;
    const int r0 = (int)min((int64_t)warp * run, (int64_t)size), r1 = (int)min((int64_t)r0 + run, (int64_t)size);
    int gt = 0, eq = 0;
    for (int i = r0 + 4 * lane; i < r1; i += 128) {
        const uint4 k = four(i);
        gt += (k.x > prefix) + (k.y > prefix) + (k.z > prefix) + (k.w > prefix);
        eq += (k.x == prefix) + (k.y == prefix) + (k.z == prefix) + (k.w == prefix);
    }
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) {
        warp_gt[warp] = gt;
        warp_eq[warp] = eq;
    }
    __syncthreads();
    const int gt_all = __reduce_add_sync(0xffffffffu, warp_gt[lane]);
    const int eq_all = __reduce_add_sync(0xffffffffu, warp_eq[lane]);
    if (t == 0) {
        mine[0] = gt_all;
        mine[1] = eq_all;
    }
    cluster.sync();
    gt = eq = 0;
    if (lane < rank) {
        const int* other = cluster.map_shared_rank(mine, lane);
        gt = other[0];
        eq = other[1];
    }
    gt = __reduce_add_sync(0xffffffffu, gt + (lane < warp ? warp_gt[lane] : 0));
    eq = __reduce_add_sync(0xffffffffu, eq + (lane < warp ? warp_eq[lane] : 0));
    for (int k0 = r0; k0 < r1; k0 += 128) {
        const int i = k0 + 4 * lane;
        const uint4 k = i < r1 ? four(i) : make_uint4(0, 0, 0, 0);
        const int g4 = (k.x > prefix) + (k.y > prefix) + (k.z > prefix) + (k.w > prefix);
        const int e4 = (k.x == prefix) + (k.y == prefix) + (k.z == prefix) + (k.w == prefix);
        const int both = g4 | e4 << 16, before = warp_sum_before(both);
        int g = gt + (before & 0xffff), e = eq + (before >> 16);
        auto put = [&](uint32_t key, int at) {
            const bool is_eq = key == prefix;
            if (key > prefix || (is_eq && e < left)) kept[g + min(e, left)] = i0 + at;
            g += key > prefix;
            e += is_eq;
        };
        put(k.x, i);
        put(k.y, i + 1);
        put(k.z, i + 2);
        put(k.w, i + 3);
        const int sums = __shfl_sync(0xffffffffu, before + both, 31);
        gt += sums & 0xffff;
        eq += sums >> 16;
    }
    cluster.sync();             // no CTA leaves while another may read its shared memory
}

constexpr int kMoveBlock = 256;

// Moves the kept rows of one KV head (blockIdx.y) of one sequence (blockIdx.z): a thread
// has one 16-byte vector of K and of V of one row, both loaded before either is stored.
template <typename T, int E>
__global__ void __launch_bounds__(kMoveBlock) evict_move(EvictArgs a) {
    constexpr int VEC = 16 / sizeof(T), NV = E / VEC, PER = kMoveBlock / NV;
    wait_before();
    const int64_t b = blockIdx.z;
    const int64_t row = b * a.KH + blockIdx.y;
    const int e = threadIdx.x % NV * VEC, at = blockIdx.x * PER + threadIdx.x / NV;
    const int slot = at < a.budget ? a.kept[row * a.budget + at] : -1;
    if (slot < 0) return;
    if (e == 0) a.new_weights[row * a.new_slots + at] = a.weights[row * a.c.slots + slot];
    const int64_t ho = blockIdx.y * a.c.head_stride + e;
    const int64_t from = a.c.offset(a.c.table + b * a.c.max_pages, slot);
    if (from < 0) return;
    const int64_t to = a.c.offset(a.new_table + b * a.new_max_pages, at);
    const Vec<T, VEC> x = ldg_stream<T, VEC>(static_cast<const T*>(a.k_cache) + from + ho);
    const Vec<T, VEC> y = ldg_stream<T, VEC>(static_cast<const T*>(a.v_cache) + from + ho);
    if (to < 0) return;
    st_stream<T, VEC>(static_cast<T*>(a.k_cache) + to + ho, x);
    st_stream<T, VEC>(static_cast<T*>(a.v_cache) + to + ho, y);
}

int launch_select(const EvictArgs& a, cudaStream_t s) {
    // More CTAs for a row while each has over 8192 slots and the GPU has SMs for them: one
    // sequence of 131067 (8 rows) takes 133, 82, 39 and 33 us with 1, 2, 4 and 8, but 16 of up
    // to 8192 (128 rows) 60, 62, 72 and 97.
    int C = 1;
    while (C < kMostCtas && a.c.slots / C > 8192 && a.B * a.KH * C * 2 <= num_sms()) C *= 2;
    const int most_keys = std::min(kMostKeys, ((a.c.slots + C - 1) / C + 3) & ~3);      // whole fours
    const size_t bytes = kHistBytes + sizeof(uint32_t) * (size_t)most_keys;
    // 48 KB, the kernel's own arrays included, need no leave; what is set is the most it can
    // ask for, so that calls of several threads do not take it from one another
    if (bytes > 32 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(evict_select, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)(kHistBytes + sizeof(uint32_t) * kMostKeys));
        if (e != cudaSuccess) {
            cudaGetLastError();
            return fail(NNOP_ERR_CUDA, std::string("paged_evict: ") + cudaGetErrorString(e));
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.B * a.KH * C));
    cfg.blockDim = dim3(kSelectThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)C, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, evict_select, a, most_keys);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(NNOP_ERR_CUDA, std::string("paged_evict: ") + cudaGetErrorString(e));
    }
    return NNOP_OK;
}

template <typename T, int E>
int launch_evict(const EvictArgs& a, cudaStream_t s) {
    constexpr int kRows = kMoveBlock / (E / (16 / (int)sizeof(T)));      // per block
    if (const int rc = launch_select(a, s)) return rc;
    if (a.budget == 0) return NNOP_OK;
    const unsigned grid = (unsigned)((a.budget + kRows - 1) / kRows);
    return launch_dependent("paged_evict", evict_move<T, E>, dim3(grid, a.KH, (unsigned)a.B), dim3(kMoveBlock), 0, s, a);
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
        if (T < 0 || QH < 0 || QH > 65535) return fail(NNOP_ERR_SHAPE, "paged_append: invalid dimensions");
        const int64_t most = ((int64_t)1 << 31) - 1024;
        if (T > most || B * T > most) return fail(NNOP_ERR_SHAPE, "paged_append: more than 2^31 - 1024 new rows");
        if ((cos_t != nullptr) != (sin_t != nullptr) || (QH == 0 && q) ||
            (QH > 0 && T > 0 && B > 0 && (!q || !q_out || !cos_t)))
            return fail(NNOP_ERR_ARG, "paged_append: cos and sin come together, and q (QH > 0) with them");
        if (cos_t && cos_batch != B && cos_batch != 1)
            return fail(NNOP_ERR_SHAPE, "paged_append: cos/sin batch must equal the batch or be 1");
        if (B == 0) return NNOP_OK;
        if (!new_lengths || new_lengths == lengths || new_lengths == n_new || (T > 0 && (!k || !v)) ||
            (pages > 0 && (!k_cache || !v_cache)))
            return fail(NNOP_ERR_ARG, "paged_append: NULL pointer, or new_lengths is lengths or n_new");
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
        a.T = paged::FastDiv((uint32_t)std::max<int64_t>(T, 1));
        a.tokens = B * T;
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
        const int64_t most = paged::kMostEvictSlots;
        if (new_max_pages < 0 || new_max_pages > most || new_max_pages * page_size > most || a.c.slots > most)
            return fail(NNOP_ERR_SHAPE, "paged_evict: more than 2^31 - 8192 slots per sequence");
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
