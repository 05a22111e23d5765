// Paged key-value cache: addressing of the page pools and the split of a ragged
// batch over the CTAs of one launch, shared by the paged_* kernels.
//
// A pool is [pages][KH][page_size][E] (any strides with E contiguous); slot j of
// sequence b lies in row j mod page_size of page table[b][j / page_size].  A table
// entry outside [0, pages) is no page: its slots are never read or written.
#pragma once

#include "common.cuh"

#include <algorithm>
#include <utility>

namespace nnop {
namespace paged {

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31 by a multiplication: the round-up method of
// Granlund and Montgomery, "Division by Invariant Integers using Multiplication" (1994),
// m = floor(2^32·(2^s − d)/d) + 1 with s = ceil(log2 d).
struct FastDiv {
    uint32_t d = 1, m = 1;
    int s = 0;
    FastDiv() = default;
    __host__ FastDiv(uint32_t div) : d(div) {
        while (s < 31 && (1u << s) < div) ++s;
        m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << s) - div)) / div + 1);
    }
    __host__ __device__ __forceinline__ uint32_t div(uint32_t n) const {
        return ((uint32_t)(((uint64_t)m * n) >> 32) + n) >> s;
    }
};

struct Cache {
    const int* table;      // [B][max_pages]
    const int* lengths;    // [B]
    uint32_t pages;
    int64_t max_pages;
    int64_t page_stride, head_stride, row_stride;   // elements
    int slots;             // max_pages · page_size, the most a sequence can hold
    FastDiv page_size;

    // Tokens sequence b has cached: its length within [0, slots].
    __device__ __forceinline__ int length(int64_t b) const { return min(max(lengths[b], 0), slots); }
    // A slot's entry in the table (0 <= slot < slots), and its row in that page.
    __device__ __forceinline__ uint32_t entry(const int* row_of_table, int slot, int& row) const {
        const uint32_t i = page_size.div((uint32_t)slot);
        row = (int)((uint32_t)slot - i * page_size.d);
        return (uint32_t)__ldg(row_of_table + i);
    }
    // Element offset of a slot's row in a head's part of the pool; negative where there is
    // no page.
    __device__ __forceinline__ int64_t offset(uint32_t page, int row) const {
        return page < pages ? page * page_stride + row * row_stride : -1;
    }
    __device__ __forceinline__ int64_t offset(const int* row_of_table, int slot) const {
        int row;
        const uint32_t page = entry(row_of_table, slot, row);
        return offset(page, row);
    }
};

// Host-side checks of what every paged entry point is given; fills `c`.
int check_cache(const char* who, Cache& c, const int32_t* table, const int32_t* lengths, int64_t E, int64_t KH,
                int64_t B, int64_t pages, int64_t page_size, int64_t max_pages, int64_t page_stride,
                int64_t head_stride, int64_t row_stride, int dtype);

// Runs an entry point's body; no C++ exception leaves the C ABI.
template <typename F>
int guarded(const char* who, F&& body) {
    try {
        return body();
    } catch (...) {
        try {
            return fail(NNOP_ERR_ARG, std::string(who) + ": out of host memory");
        } catch (...) {
            return NNOP_ERR_ARG;
        }
    }
}

// ---------------------------------------------------------------------------
// Split of a ragged batch.  The work of one launch is a list of units: for every
// sequence b (in order), for every head tile h < heads, the sequence's chunks of
// `unit` slots.  CTA c of G = min(CTAs launched, units) takes units [start(c),
// start(c + 1)), start(c) = floor(units·c / G), so all CTAs get the same number of
// units (to one) whatever the lengths are -- they live on the device, the host never
// sees them -- and none is without one.  A CTA walks its units as segments:
// consecutive chunks of one (b, h).
//
// To begin and end a segment costs a CTA time too, so where CTAs have several units each
// every (b, h) counts `kExtra` units more, empty ones in front (extra).  A CTA whose share
// of a (b, h) is empty units alone leaves them to the next CTA.
// ---------------------------------------------------------------------------
constexpr int kThreads = 128;

// n / d of numbers that mostly fit 32 bits.
__host__ __device__ __forceinline__ long long div_small(long long n, long long d) {
    if (((unsigned long long)(n | d) >> 32) == 0) return (uint32_t)n / (uint32_t)d;
    return n / d;
}

struct SplitShared {
    long long chunks[kThreads / 32];
    int some[kThreads / 32];
    long long before;
    int b;
};

struct Split {
    long long units;       // over all sequences and head tiles
    long long u, u1;       // this CTA's units left
    int G;                 // CTAs with units
    int extra;             // empty chunks in front of every (b, h)
    int b, h, chunk, chunks, len;
    long long before;      // units / heads in front of sequence b

    __host__ __device__ __forceinline__ static long long start(long long units, int c, int G) {
        return div_small(units * c, G);
    }
    // The CTA that has unit e: the largest c with start(c) <= e.
    __host__ __device__ __forceinline__ int owner(long long e) const {
        return (int)div_small((e + 1) * G + units - 1, units) - 1;
    }
    template <int kUnit>
    __device__ __forceinline__ int chunks_of(int n) const {
        return n == 0 ? 0 : (n + kUnit - 1) / kUnit + extra;
    }
    // One past this CTA's last chunk of (b, h); 0: no segment is left.
    __device__ __forceinline__ int segment() const {
        if (u >= u1) return 0;
        const int c1 = (int)min((long long)chunks, chunk + (u1 - u));
        return c1 <= extra && c1 < chunks ? 0 : c1;
    }
    // Slots [first, end) of chunks c0 to c1 - 1 of this sequence.
    template <int kUnit>
    __device__ __forceinline__ int first_slot(int c0) const { return max(c0 - extra, 0) * kUnit; }
    template <int kUnit>
    __device__ __forceinline__ int end_slot(int c1) const { return min(len, (c1 - extra) * kUnit); }
};

// Block-wide (kThreads threads): the units as `ctas` CTAs share them (extra, G), and
// part `index` of `parts` of them, set to its first unit.
template <int kUnit, int kExtra>
__device__ __forceinline__ Split split_begin(const Cache& c, int64_t B, int heads, int ctas, int index, int parts,
                                             SplitShared& sh) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int64_t per = (B + kThreads - 1) / kThreads;
    const int64_t b0 = min((int64_t)t * per, B), b1 = min(b0 + per, B);
    long long mine = 0;
    int some = 0;              // sequences with slots
    for (int64_t b = b0; b < b1; ++b) {
        const int n = c.length(b);
        mine += (n + kUnit - 1) / kUnit;
        some += n > 0;
    }
    long long incl = mine;
    int incl_some = some;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, incl, o);
        const int up_some = __shfl_up_sync(0xffffffffu, incl_some, o);
        if (lane >= o) {
            incl += up;
            incl_some += up_some;
        }
    }
    if (lane == 31) {
        sh.chunks[warp] = incl;
        sh.some[warp] = incl_some;
    }
    __syncthreads();
    long long before = incl - mine, total = 0;
    int before_some = incl_some - some, total_some = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) {
            before += sh.chunks[w];
            before_some += sh.some[w];
        }
        total += sh.chunks[w];
        total_some += sh.some[w];
    }
    Split s;
    s.extra = total * heads > ctas ? kExtra : 0;
    before += s.extra * before_some;
    mine += s.extra * some;
    s.units = (total + (long long)s.extra * total_some) * heads;
    s.G = (int)min((long long)ctas, s.units);
    s.u = s.u1 = 0;
    parts = (int)min((long long)parts, s.units);
    if (index < parts) {
        s.u = Split::start(s.units, index, parts);
        s.u1 = Split::start(s.units, index + 1, parts);
    }
    if (s.u < s.u1) {
        const long long x = div_small(s.u, heads);      // in sequence b: before(b) <= x < before(b) + chunks(b)
        if (x >= before && x < before + mine) {
            int64_t b = b0;
            for (;; ++b) {
                const int n = s.chunks_of<kUnit>(c.length(b));
                if (x < before + n) break;
                before += n;
            }
            sh.b = (int)b;
            sh.before = before;
        }
        __syncthreads();
        s.b = sh.b;
        s.before = sh.before;
        s.len = c.length(s.b);
        s.chunks = s.chunks_of<kUnit>(s.len);
        const long long r = s.u - s.before * heads;
        s.h = (int)div_small(r, s.chunks);
        s.chunk = (int)(r - (long long)s.h * s.chunks);
        if (s.chunk <= s.extra) {
            s.u -= s.chunk;
            s.chunk = 0;
        }
    }
    return s;
}

// On from the segment that ended at chunk c1.
template <int kUnit>
__device__ __forceinline__ void split_next(Split& s, int c1, const Cache& c, int heads) {
    s.u += c1 - s.chunk;
    s.chunk = 0;
    if (s.u >= s.u1 || ++s.h < heads) return;
    s.h = 0;
    do {
        s.before += s.chunks;
        s.len = c.length(++s.b);
        s.chunks = s.chunks_of<kUnit>(s.len);
    } while (s.chunks == 0);
}

// Launch that may start while the kernel in front of it in the stream drains; the
// kernel calls wait_before() before it touches that kernel's results.
template <typename... KArgs, typename... Args>
int launch_dependent(const char* what, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                     cudaStream_t s, Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(NNOP_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
    }
    return NNOP_OK;
}
__device__ __forceinline__ void wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace paged
}  // namespace nnop
