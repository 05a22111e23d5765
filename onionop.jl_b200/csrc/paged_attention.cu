// Attention of one new token per sequence over a paged key-value cache:
//   s_j = scale·(q · k_j),  o = Σ_j softmax(s)_j v_j,  lse = log Σ_j exp(s_j)
// over the slots j < lengths[b] that have a page, every query head of a KV head's
// group reading the same rows.  Optionally weights[b][kv head][j] += Σ over the
// group's heads of softmax(s)_j, which is what nnop_paged_evict goes by.
//
// Bound: HBM.  Each cached row is read once for all query heads of its group, 2·Σ
// lengths·KH·E·size bytes, against 4·Σ lengths·QH·E flops, where the group fits a head
// tile of R heads: 8, 16 or 32 in 16 bits, 1 to 8 in fp32 (rows_per_tile).  A larger
// group's rows are read once per tile, ceil(group / R) times; with tiles of 32 the two
// warps of a key group each load them, the second time mostly from L2.
//
// Times in this file are of CUDA events around calls queued behind one another.
//
// One launch splits the batch evenly over its CTAs whatever the lengths are
// (paged.cuh).  A CTA runs a softmax over its part of a sequence with a running
// maximum and sum, every warp on keys of its own, and joins its warps through
// shared memory.  A (sequence, head tile) that lies in one CTA is written at once;
// the others leave (maximum, sum, accumulator) in the workspace and a second launch
// joins them.  The weights need the final maximum and sum, so the scores are kept
// (fp32, workspace) and the second launch turns them into weights: 8 bytes per (query
// head, slot) instead of reading K again (E·size).
#include "paged.cuh"

#include <cmath>
#include <type_traits>

namespace nnop {
namespace paged {
namespace {

constexpr int kMaxCtas = 444;      // 148 SMs × 3; the workspace is sized for it
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnArgs {
    const void *q, *k, *v;
    void* o;
    float *lse, *weights;
    Cache c;
    int64_t B;
    int QH, KH, group, tiles;      // tiles: head tiles of R rows per KV head
    float scale2;                  // scale · log2(e)
    int4* join;                    // [kMaxCtas] (b, head tile, CTAs, -) of a split that starts in CTA c; CTAs = 0: none
    float2* part_ml;               // [2·kMaxCtas][R] maximum (scaled, log2 domain), sum of exp2(s·scale2 − maximum)
    float* part_acc;               // [2·kMaxCtas][R][E]
    float* scores;                 // [B][QH][slots] q·k, unscaled (with weights)
    float2* row_ml;                // [B][QH] as part_ml, of a row that lies in one CTA (with weights)
};

// For what ends in 16 bits: exp2f without its results below 2^-126 (0 here), of weights
// whose largest is 1.  fp32 and the weights' sums take exp2f, which has them.
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A sequence without a single score: zeros, lse −Inf.
template <typename T, int E>
__device__ __forceinline__ void write_row(const AttnArgs& a, int64_t b, int qh, int e, float acc, float m, float l) {
    const int64_t row = b * a.QH + qh;
    static_cast<T*>(a.o)[row * E + e] = from_f<T>(l > 0.f || l != l ? acc / l : 0.f);
    if (e == 0) {
        a.lse[row] = l > 0.f || l != l ? (m + log2f(l)) * kLn2 : -INFINITY;
        if (a.row_ml != nullptr) a.row_ml[row] = make_float2(m, l);
    }
}

// Sequences of length 0 have no unit: their rows are written here.
template <typename T, int E>
__device__ __forceinline__ void write_empty(const AttnArgs& a) {
    for (int64_t b = blockIdx.x; b < a.B; b += gridDim.x) {
        if (a.c.length(b) != 0) continue;
        for (int i = threadIdx.x; i < a.QH * E; i += kThreads) write_row<T, E>(a, b, i / E, i % E, 0.f, 0.f, 0.f);
    }
}

// What stands for a row that is not there: a finite V, so that its weight of 0 counts.
__device__ const uint4 no_row[16] = {};

template <int E> struct SimtShape {
    static constexpr int kGroups = E >= 128 ? 1 : E == 64 ? 2 : 4;   // of 8 keys that a warp takes at once (8 KB of K and V from E = 32)
    static constexpr int kUnit = 8 * kGroups;                        // slots per unit of the split
};
constexpr int kSimtExtra = 8;      // units that a segment's begin and end cost (as in attention_mma)

// fp32 (no tensor cores: their formats would cost its accuracy): a quad of lanes per key
// for the scores, E/32 columns per lane for the products with V, R query heads per pass
// over the keys.  A step's rows are all in flight before any is used, K of the next step
// while this one's softmax runs, V while the next scores do: 107 us (16 sequences up to
// 8192, 32/8 heads of 128, 538 MB); loads under a branch, one at a time, took 259.
template <int E, int R>
__global__ void __launch_bounds__(kThreads, 3)
attention_simt(AttnArgs a) {
    constexpr int NQ = E >= 16 ? E / 16 : 1;          // 16-byte vectors per lane of a quad
    constexpr int COLS = E >= 32 ? E / 32 : 1;        // columns per lane
    constexpr int KG = SimtShape<E>::kGroups, kKeys = 8 * KG, kUnit = SimtShape<E>::kUnit;
    __shared__ SplitShared sh;
    __shared__ __align__(16) float qs[R][E];
    __shared__ float wm[4][R], wl[4][R], wacc[4][R][E];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, sub = lane & 3;
    const int heads = a.KH * a.tiles;
    let_next_start();
    Split s = split_begin<kUnit, kSimtExtra>(a.c, a.B, heads, gridDim.x, blockIdx.x, gridDim.x, sh);
    write_empty<float, E>(a);
    if (threadIdx.x == 0) a.join[blockIdx.x] = make_int4(0, 0, 0, 0);
    while (const int c1 = s.segment()) {
        const int c0 = s.chunk;
        const int kvh = s.h / a.tiles, r0 = (s.h % a.tiles) * R;
        const int rows = min(R, a.group - r0);
        const int qh0 = kvh * a.group + r0;
        const int* tab = a.c.table + (int64_t)s.b * a.c.max_pages;
        const float* K = static_cast<const float*>(a.k) + kvh * a.c.head_stride;
        const float* V = static_cast<const float*>(a.v) + kvh * a.c.head_stride;
        const float* none = reinterpret_cast<const float*>(no_row);
        for (int i = threadIdx.x; i < R * E; i += kThreads)
            qs[i / E][i % E] = i / E < rows ? static_cast<const float*>(a.q)[((int64_t)s.b * a.QH + qh0) * E + i] : 0.f;
        __syncthreads();
        float m[R], l[R], acc[R][COLS];      // m: maximum of the unscaled scores
#pragma unroll
        for (int r = 0; r < R; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
#pragma unroll
            for (int i = 0; i < COLS; ++i) acc[r][i] = 0.f;
        }
        const int end = s.end_slot<kUnit>(c1);
        constexpr int kStep = 4 * kKeys;
        float4 kr[KG][NQ];
        float vr[KG][8][COLS];
        int64_t off[KG];               // of this quad's keys; negative: no row
        auto load_k = [&](int64_t (&o)[KG], int key0) {
#pragma unroll
            for (int g = 0; g < KG; ++g) {
                const int key = key0 + g * 8 + quad;
                o[g] = key < end ? a.c.offset(tab, key) : -1;
                const float* p = o[g] >= 0 ? K + o[g] + sub * 4 : none;
#pragma unroll
                for (int i = 0; i < NQ; ++i) kr[g][i] = __ldcs(reinterpret_cast<const float4*>(p + (o[g] >= 0 ? i * 16 : 0)));
            }
        };
        auto load_v = [&](const int64_t (&o)[KG]) {
#pragma unroll
            for (int g = 0; g < KG; ++g)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int64_t x = __shfl_sync(0xffffffffu, o[g], j * 4);
                    const float* p = x >= 0 && lane * COLS < E ? V + x + lane * COLS : none;
                    load_vec<float, COLS>(vr[g][j], p);
                }
        };
        int key0 = s.first_slot<kUnit>(c0) + warp * kKeys;
        if (key0 < end) {
            load_k(off, key0);
            load_v(off);
        }
        for (; key0 < end; key0 += kStep) {
            float sc[KG][R];
#pragma unroll
            for (int g = 0; g < KG; ++g)
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float dot = 0.f;
#pragma unroll
                    for (int i = 0; i < NQ; ++i) {
                        const float4 x = *reinterpret_cast<const float4*>(&qs[r][(i * 4 + sub) * 4]);
                        dot = fmaf(kr[g][i].x, x.x, dot);
                        dot = fmaf(kr[g][i].y, x.y, dot);
                        dot = fmaf(kr[g][i].z, x.z, dot);
                        dot = fmaf(kr[g][i].w, x.w, dot);
                    }
                    sc[g][r] = dot;
                }
            const bool more = key0 + kStep < end;
            int64_t here[KG];
#pragma unroll
            for (int g = 0; g < KG; ++g) here[g] = off[g];
            if (more) load_k(off, key0 + kStep);
#pragma unroll
            for (int g = 0; g < KG; ++g)
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float x = sc[g][r];
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    x += __shfl_xor_sync(0xffffffffu, x, 2);
                    sc[g][r] = here[g] >= 0 ? x : -INFINITY;
                }
            if (a.scores != nullptr && sub == 0) {
#pragma unroll
                for (int g = 0; g < KG; ++g)
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const int key = key0 + g * 8 + quad;
                        if (key < end && r < rows)
                            a.scores[((int64_t)s.b * a.QH + qh0 + r) * a.c.slots + key] = sc[g][r];
                    }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float mx = sc[0][r];
#pragma unroll
                for (int g = 1; g < KG; ++g) mx = fmaxf(mx, sc[g][r]);
                // the maximum rises only now and then: the lanes meet only when one of them has more
                if (__any_sync(0xffffffffu, mx > m[r])) {
                    mx = fmaxf(mx, m[r]);
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                    const float alpha = exp2f(__fmul_rn(m[r], a.scale2) - __fmul_rn(mx, a.scale2));
                    m[r] = mx;
                    l[r] *= alpha;
#pragma unroll
                    for (int i = 0; i < COLS; ++i) acc[r][i] *= alpha;
                }
                const float base = m[r] == -INFINITY ? 0.f : __fmul_rn(m[r], a.scale2);      // -Inf: no score yet
#pragma unroll
                for (int g = 0; g < KG; ++g) {
                    sc[g][r] = exp2f(fmaf(sc[g][r], a.scale2, -base));
                    l[r] += sc[g][r];
                }
            }
#pragma unroll
            for (int g = 0; g < KG; ++g)
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float p = __shfl_sync(0xffffffffu, sc[g][r], j * 4);
#pragma unroll
                        for (int i = 0; i < COLS; ++i) acc[r][i] = fmaf(p, vr[g][j][i], acc[r][i]);
                    }
            if (more) load_v(off);
        }
        // join the warps
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
            if (lane == 0) {
                wm[warp][r] = __fmul_rn(m[r], a.scale2);
                wl[warp][r] = l[r];
            }
            if (lane * COLS < E) {
#pragma unroll
                for (int i = 0; i < COLS; ++i) wacc[warp][r][lane * COLS + i] = acc[r][i];
            }
        }
        __syncthreads();
        const bool whole = c0 == 0 && c1 == s.chunks;
        const int slot = 2 * blockIdx.x + (c0 == 0 ? 1 : 0);
        for (int i = threadIdx.x; i < rows * E; i += kThreads) {
            const int r = i / E, e = i % E;
            const float mx = fmaxf(fmaxf(wm[0][r], wm[1][r]), fmaxf(wm[2][r], wm[3][r]));
            const float base = mx == -INFINITY ? 0.f : mx;
            float sum = 0.f, ac = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = exp2f(wm[w][r] - base);
                sum = fmaf(wl[w][r], f, sum);
                ac = fmaf(wacc[w][r][e], f, ac);
            }
            if (whole) {
                write_row<float, E>(a, s.b, qh0 + r, e, ac, mx, sum);
            } else {
                a.part_acc[((int64_t)slot * R + r) * E + e] = ac;
                if (e == 0) a.part_ml[slot * R + r] = make_float2(mx, sum);
            }
        }
        if (!whole && c0 == 0 && threadIdx.x == 0)
            a.join[blockIdx.x] = make_int4(s.b, s.h, s.owner(s.u + s.chunks - 1) - blockIdx.x + 1, 0);
        split_next<kUnit>(s, c1, a.c, heads);
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Tensor-core kernel for the 16-bit types (mma.sync m16n8k16).  The op is bound by
// HBM (with up to 8 query heads a key row the tensor pipe is busy 15% of the time),
// so what matters is that the loads never stop, and the operands go from global
// memory straight into the fragments -- no shared memory, no barrier, every warp on its own keys:
//
//   Sᵀ (16 keys × 8 heads) = K (A: 16 × E) · Qᵀ (B: E × 8)
//   Oᵀ (E × 8 heads)      += Vᵀ (A: E × 16 keys) · Pᵀ (B: 16 keys × 8)
//
// with keys (then E) on the side of 16 and the group's heads on the side of 8, so a
// group of up to 8 heads wastes nothing.  A sum over E may run in any order, so a
// lane's A fragments of two k16 steps are the 16 consecutive bytes it loads of a K
// row (4 lanes read 64 bytes of each of 8 rows), and Q is laid out to match.  The
// rows of Oᵀ may be any E order too: a lane loads 16 bytes of 4 V rows (8 lanes read
// 128 bytes of a row) and pairs two keys' halves by byte permutes.  Sᵀ's
// accumulators become Pᵀ's B fragments by movmatrix.  P keeps fp32's bits, to ex2's own
// error of 2^-22: it goes in as the sum of three bf16 terms or two f16 terms (pack2).
// Rounded once to 16 bits it would cost as much accuracy as rounding the result does; of
// 65536 bf16 results (16 sequences up to 8192) two terms rounded 78 to another side than
// exact values do, three 51, products in fp32 34.  The third term takes 64 sequences up to
// 8192 with 16 heads a group from 111 to 117 us; 4 heads stay at 169 (the launch alone).
// f16: P is scaled by 2^14, which the running sum shares, so that weights down to 2^-38 of
// the largest count.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}

// W words of a row that is read once.
template <int W>
__device__ __forceinline__ void load_words(uint32_t (&r)[W], const char* p) {
    if constexpr (W == 4)
        asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "l"(p));
    else if constexpr (W == 2)
        asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "l"(p));
    else
        asm volatile("ld.global.nc.L1::no_allocate.b32 %0, [%1];" : "=r"(r[0]) : "l"(p));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Two values as a pair of T, rounded to nearest or (kRest) towards zero with what that
// left of them in their place.  The rest of a value above 0 is above 0 too, so that an
// infinite element of V times each of a probability's terms has one sign: bf16 makes the
// rest larger by 2^-23 of the probability for that, f16 at least its smallest number, 2^-24
// (2^-38 of the largest probability).
template <typename T, bool kRest, int kTerm>
__device__ __forceinline__ uint32_t pack2(float& lo, float& hi) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) {
        if constexpr (!kRest) {
            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
            return r;
        }
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        const __half2 h = *reinterpret_cast<const __half2*>(&r);
        lo = fmaxf(lo - __low2float(h), fminf(__low2float(h), 0x1p-24f));
        hi = fmaxf(hi - __high2float(h), fminf(__high2float(h), 0x1p-24f));
    } else {
        if constexpr (!kRest) {
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
            return r;
        }
        asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        // the first rest is up to 2^-7 of the probability
        constexpr float kMore = kTerm == 0 ? 1.f + 0x1p-23f : 1.f + 0x1p-16f;
        lo = fmaf(lo, kMore, -__uint_as_float(r << 16));
        hi = fmaf(hi, kMore, -__uint_as_float(r & 0xffff0000u));
    }
    return r;
}

template <int E> struct MmaShape {
    static constexpr int kTiles = E >= 128 ? 1 : E == 64 ? 2 : 4;   // 16-key tiles a warp takes at once (8 KB of K and V from E = 32)
    static constexpr int kKeys = 16 * kTiles;
    static constexpr int kUnit = kKeys;                             // slots per unit of the split
};

// CTAs per SM.  What has to be in flight to keep HBM busy lies in registers, 8 KB a
// warp, beside 32·NT for Oᵀ and 16·NT for Q: three CTAs of 168 registers a thread, which
// spill 24 bytes at most (170 us for 64 sequences up to 8192, heads of 64 91 us, of 32 57),
// before two of 255 (177, 99, 66) or four of 128, which spill all they hold (216, 94, 58);
// with two head tiles a warp, two.  A ring in shared memory filled by cp.async, with up to
// 192 KB in flight, was slower when it was tried: 173 us where this took 167, and 107
// instead of 90 for heads of 64.
constexpr int mma_ctas(int NT) { return NT == 1 ? 3 : 2; }
// What a segment's begin and end count for, in units (8 KB; a CTA among two has a larger
// share of HBM than one among three).  64 sequences up to 8192: 2 units 179 us, 4 units
// 172, 8 units 170; 32 of them with two head tiles: 8 units 142 us, 12 units 130, 16 units
// 117, 24 units 119.
constexpr int mma_extra(int NT) { return NT == 1 ? 8 : 16; }

// NT: head tiles (of 8) per warp, which share the fragments of K and V.  WT: warps
// that read the same keys for other head tiles; 4/WT warps share the keys out.
template <typename T, int E, int NT, int WT, bool kWholeTiles>
__global__ void __launch_bounds__(kThreads, mma_ctas(NT))
attention_mma(AttnArgs a) {
    using S = MmaShape<E>;
    constexpr int R = 8 * NT * WT;
    constexpr int KW = E >= 32 ? 4 : 2, KC = E / (8 * KW);     // words per K load, loads per row
    constexpr int VW = E >= 64 ? 4 : E == 32 ? 2 : 1, VC = E / (16 * VW);
    constexpr float kShift = std::is_same<T, __half>::value ? 14.f : 0.f;
    constexpr int kTerms = std::is_same<T, __half>::value ? 2 : 3;
    __shared__ SplitShared sh;
    __shared__ float wm[4][8 * NT], wl[4][8 * NT];
    __shared__ __align__(16) float wacc[4][8 * NT][E];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gid = lane >> 2, sub = lane & 3;
    const int tile0 = warp % WT * NT, part = warp / WT;
    const int heads = a.KH * a.tiles;
    let_next_start();
    Split s = split_begin<S::kUnit, mma_extra(NT)>(a.c, a.B, heads, gridDim.x, blockIdx.x, gridDim.x, sh);
    write_empty<T, E>(a);
    if (threadIdx.x == 0) a.join[blockIdx.x] = make_int4(0, 0, 0, 0);
    int c1 = s.segment();
    if (c1 == 0) return;

    int rows, qh0, end, key0;
    const int* tab;
    uint32_t q[NT][KC][KW];        // B fragments of all k16 steps; head gid of each of this warp's tiles
    uint32_t kr[S::kTiles][2][KC][KW], vr[S::kTiles][4][VC][VW];
    const char *kl, *vl;           // this head's pools, at this lane's first row and bytes of a tile
    // Bytes between a lane's rows: K 8 rows on; V 1, 8 and 9 rows on.
    const int64_t rs = a.c.row_stride * 2;
    const bool odd_pages = a.c.page_size.d & 1;
    constexpr int kStep = S::kKeys * (4 / WT);

    // Where a step's rows are.  kWholeTiles (pages of a multiple of 16 slots): a tile of 16
    // keys lies in one page, one lookup for all lanes, its table entry fetched a step ahead
    // (fetched with the rows it took 175 us instead of 168 for 64 sequences up to 8192).  Else
    // one lookup for each row a lane reads (pages of 20: 171 us as against 170, but heads of
    // 64 in pages of 16 would take 111 us that way instead of 91, heads of 32 96 instead of 57).
    uint32_t page[S::kTiles];      // table entries of the next step's tiles
    int row[S::kTiles];
    int64_t tiles[S::kTiles] = {}; // bytes into the pool; negative: no page
    bool inside;                   // all of the step's keys have rows
    auto find = [&](int key0) {
        if constexpr (kWholeTiles) {
#pragma unroll
            for (int t = 0; t < S::kTiles; ++t)
                page[t] = key0 + t * 16 < end ? a.c.entry(tab, key0 + t * 16, row[t]) : ~0u;
        }
    };
    auto found = [&](int key0) {
        inside = kWholeTiles && key0 + S::kKeys <= end;
        if constexpr (kWholeTiles) {
#pragma unroll
            for (int t = 0; t < S::kTiles; ++t) {
                tiles[t] = a.c.offset(page[t], row[t]) * 2;
                inside = inside && tiles[t] >= 0;
            }
        }
    };
    // Bytes into the pool of key + mine of tile t, counted from where kl and vl point.
    auto row_at = [&](int t, int key, int mine, int first) -> int64_t {
        if (key + mine >= end) return -1;
        if constexpr (kWholeTiles) return tiles[t] < 0 ? -1 : tiles[t] + (mine - first) * rs;
        const int64_t x = a.c.offset(tab, key + mine);
        return x < 0 ? -1 : x * 2;
    };
    // Where a lane reads K of tile t, rows gid and 8 + gid; bit 2t + i of has: there is a row.
    auto k_rows = [&](const char* (&p)[2], int t, int key0, uint32_t& has) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t x = row_at(t, key0 + t * 16, i * 8 + gid, gid);
            if (x < 0) has &= ~(1u << (2 * t + i));
            p[i] = x >= 0 ? kl + x : reinterpret_cast<const char*>(no_row);
        }
    };
    // ... and V of tile t, rows 2·sub, 2·sub + 1 and both 8 on.
    auto v_rows = [&](const char* (&p)[4], int t, int key0) {
        int64_t x = -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int mine = (i >> 1) * 8 + (i & 1) + 2 * sub;
            // pages of an even number of slots hold both keys of a pair
            if (kWholeTiles || i % 2 == 0 || odd_pages) x = row_at(t, key0 + t * 16, mine, 2 * sub);
            else x = x < 0 || key0 + t * 16 + mine >= end ? -1 : x + rs;
            p[i] = x >= 0 ? vl + x : reinterpret_cast<const char*>(no_row);
        }
    };
    auto load_k = [&](int key0, uint32_t& has) {
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) {
            const char* p[2] = {};
            if (!inside) k_rows(p, t, key0, has);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int c = 0; c < KC; ++c)
                    load_words<KW>(kr[t][i][c], (inside ? kl + tiles[t] + i * 8 * rs : p[i]) + c * (16 * KW));
        }
    };
    auto load_v = [&](int key0) {
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) {
            const char* p[4] = {};
            if (!inside) v_rows(p, t, key0);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < VC; ++c)
                    load_words<VW>(vr[t][i][c],
                                   (inside ? vl + tiles[t] + ((i >> 1) * 8 + (i & 1)) * rs : p[i]) + c * (32 * VW));
        }
    };
    uint32_t live = 0;
    // The segment [s.chunk, c1) of (s.b, s.h): its Q, and the first step's K and V.
    auto enter = [&]() {
        const int kvh = s.h / a.tiles, r0 = (s.h - kvh * a.tiles) * R;
        rows = min(R, a.group - r0);
        qh0 = kvh * a.group + r0;
        tab = a.c.table + (int64_t)s.b * a.c.max_pages;
        kl = static_cast<const char*>(a.k) + kvh * a.c.head_stride * 2 + sub * (4 * KW) + (kWholeTiles ? gid * rs : 0);
        vl = static_cast<const char*>(a.v) + kvh * a.c.head_stride * 2 + gid * (4 * VW) + (kWholeTiles ? 2 * sub * rs : 0);
        end = s.end_slot<S::kUnit>(c1);
        key0 = s.first_slot<S::kUnit>(s.chunk) + part * S::kKeys;
        find(key0);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = (tile0 + n) * 8 + gid;
            const char* row = r < rows ? static_cast<const char*>(a.q) + ((int64_t)s.b * a.QH + qh0 + r) * (2 * E) + sub * (4 * KW)
                                       : reinterpret_cast<const char*>(no_row);
#pragma unroll
            for (int c = 0; c < KC; ++c) load_words<KW>(q[n][c], row + c * (16 * KW));
        }
        if (key0 < end) {
            found(key0);
            live = ~0u;
            load_k(key0, live);
            load_v(key0);
            find(key0 + kStep);
        }
    };
    enter();
    for (;;) {
        // running maximum of the raw scores of heads 2·sub and 2·sub + 1, what the weights are
        // relative to (log2), this lane's sum of weights, Oᵀ
        float m[NT][2], base[NT][2], l[NT][2], acc[NT][VC][VW][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                m[n][j] = -INFINITY;
                base[n][j] = l[n][j] = 0.f;
            }
#pragma unroll
            for (int c = 0; c < VC; ++c)
#pragma unroll
                for (int j = 0; j < VW; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[n][c][j][i] = 0.f;
        }
        for (; key0 < end; key0 += kStep) {
            // Pages of other sizes: each chunk's registers are loaded again as soon as its
            // products are through (pages of 20: 169 us instead of 179 when it was tried).
            const bool more = key0 + kStep < end;
            uint32_t next = ~0u;
            if (more) found(key0 + kStep);
            float d[NT][S::kTiles][4];
#pragma unroll
            for (int t = 0; t < S::kTiles; ++t) {
                const char* p[2] = {};
                if (!kWholeTiles && more) k_rows(p, t, key0 + kStep, next);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) d[n][t][i] = 0.f;
#pragma unroll
                for (int c = 0; c < KC; ++c) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int w = 0; w < KW; w += 2)
                            mma16816<T>(d[n][t], kr[t][0][c][w], kr[t][1][c][w], kr[t][0][c][w + 1], kr[t][1][c][w + 1],
                                        q[n][c][w], q[n][c][w + 1]);
                    if (!kWholeTiles && more) {
                        load_words<KW>(kr[t][0][c], p[0] + c * (16 * KW));
                        load_words<KW>(kr[t][1][c], p[1] + c * (16 * KW));
                    }
                }
            }
            if (kWholeTiles && more) load_k(key0 + kStep, next);
            if (live != ~0u) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int t = 0; t < S::kTiles; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!(live >> (2 * t + i / 2) & 1)) d[n][t][i] = -INFINITY;
            }
            if (a.scores != nullptr) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int t = 0; t < S::kTiles; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = key0 + t * 16 + i / 2 * 8 + gid, r = (tile0 + n) * 8 + 2 * sub + i % 2;
                            if (key < end && r < rows)
                                a.scores[((int64_t)s.b * a.QH + qh0 + r) * a.c.slots + key] = d[n][t][i];
                        }
            }
            uint32_t b[NT][S::kTiles][kTerms][2];      // Pᵀ: [16-bit term][key half]
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float mx[2] = {d[n][0][0], d[n][0][1]};
#pragma unroll
                for (int t = 0; t < S::kTiles; ++t) {
                    mx[0] = fmaxf(mx[0], fmaxf(d[n][t][0], d[n][t][2]));
                    mx[1] = fmaxf(mx[1], fmaxf(d[n][t][1], d[n][t][3]));
                }
                // the maximum rises only now and then: the lanes meet only when one of them has more
                if (__any_sync(0xffffffffu, mx[0] > m[n][0] || mx[1] > m[n][1])) {
                    float f[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        mx[j] = fmaxf(mx[j], m[n][j]);
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], o));
                        const float to = mx[j] == -INFINITY ? 0.f : mx[j] * a.scale2 - kShift;    // -Inf: no score yet
                        f[j] = m[n][j] == -INFINITY ? 0.f : fast_exp2(base[n][j] - to);
                        m[n][j] = mx[j];
                        base[n][j] = to;
                        l[n][j] *= f[j];
                    }
#pragma unroll
                    for (int c = 0; c < VC; ++c)
#pragma unroll
                        for (int j = 0; j < VW; ++j)
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[n][c][j][i] *= f[i & 1];
                }
#pragma unroll
                for (int t = 0; t < S::kTiles; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float p0 = fast_exp2(fmaf(d[n][t][i * 2], a.scale2, -base[n][0]));
                        float p1 = fast_exp2(fmaf(d[n][t][i * 2 + 1], a.scale2, -base[n][1]));
                        l[n][0] += p0;
                        l[n][1] += p1;
                        b[n][t][0][i] = transpose8x8(pack2<T, true, 0>(p0, p1));
                        if constexpr (kTerms == 3) b[n][t][1][i] = transpose8x8(pack2<T, true, 1>(p0, p1));
                        b[n][t][kTerms - 1][i] = transpose8x8(pack2<T, false, kTerms - 1>(p0, p1));
                    }
            }
#pragma unroll
            for (int t = 0; t < S::kTiles; ++t) {
                const char* p[4] = {};
                if (!kWholeTiles && more) v_rows(p, t, key0 + kStep);
#pragma unroll
                for (int c = 0; c < VC; ++c) {
#pragma unroll
                    for (int j = 0; j < VW; ++j) {
                        const uint32_t a0 = __byte_perm(vr[t][0][c][j], vr[t][1][c][j], 0x5410);
                        const uint32_t a1 = __byte_perm(vr[t][0][c][j], vr[t][1][c][j], 0x7632);
                        const uint32_t a2 = __byte_perm(vr[t][2][c][j], vr[t][3][c][j], 0x5410);
                        const uint32_t a3 = __byte_perm(vr[t][2][c][j], vr[t][3][c][j], 0x7632);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int k = 0; k < kTerms; ++k)
                                mma16816<T>(acc[n][c][j], a0, a1, a2, a3, b[n][t][k][0], b[n][t][k][1]);
                    }
                    if (!kWholeTiles && more) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) load_words<VW>(vr[t][i][c], p[i] + c * (32 * VW));
                    }
                }
            }
            if (kWholeTiles && more) load_v(key0 + kStep);
            live = next;
            find(key0 + 2 * kStep);
        }
        // The next segment's first loads go out before this one's warps are joined.
        const bool first = s.chunk == 0, whole = first && c1 == s.chunks;
        const int slot = 2 * blockIdx.x + (first ? 1 : 0);
        const int b_of = s.b, rows_of = rows, qh_of = qh0;
        if (!whole && first && threadIdx.x == 0)
            a.join[blockIdx.x] = make_int4(s.b, s.h, s.owner(s.u + s.chunks - 1) - blockIdx.x + 1, 0);
        split_next<S::kUnit>(s, c1, a.c, heads);
        c1 = s.segment();
        if (c1 != 0) enter();
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], o);
                if (gid == 0) {
                    wm[warp][n * 8 + 2 * sub + j] = m[n][j] == -INFINITY ? -INFINITY : base[n][j];
                    wl[warp][n * 8 + 2 * sub + j] = l[n][j];
                }
            }
#pragma unroll
            for (int c = 0; c < VC; ++c)
#pragma unroll
                for (int j = 0; j < VW; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        *reinterpret_cast<float2*>(&wacc[warp][n * 8 + 2 * sub + h][(c * 8 + gid) * (2 * VW) + 2 * j]) =
                            make_float2(acc[n][c][j][h], acc[n][c][j][2 + h]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < rows_of * E; i += kThreads) {
            const int r = i / E, e = i % E;
            float mw[4 / WT], mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < 4 / WT; ++w) {
                mw[w] = wm[w * WT + r / (8 * NT)][r % (8 * NT)];
                mx = fmaxf(mx, mw[w]);
            }
            const float base = mx == -INFINITY ? 0.f : mx;
            float sum = 0.f, ac = 0.f;
#pragma unroll
            for (int w = 0; w < 4 / WT; ++w) {
                const float f = fast_exp2(mw[w] - base);
                sum = fmaf(wl[w * WT + r / (8 * NT)][r % (8 * NT)], f, sum);
                ac = fmaf(wacc[w * WT + r / (8 * NT)][r % (8 * NT)][e], f, ac);
            }
            if (whole) {
                write_row<T, E>(a, b_of, qh_of + r, e, ac, mx, sum);
            } else {
                a.part_acc[((int64_t)slot * R + r) * E + e] = ac;
                if (e == 0) a.part_ml[slot * R + r] = make_float2(mx, sum);
            }
        }
        if (c1 == 0) return;
        __syncthreads();
    }
}

// Joins two parts of a row: maximum (log2 domain), sum and what is weighed with them.
__device__ __forceinline__ float2 join_two(float2 x, float2 y, float& fx, float& fy) {
    const float mx = fmaxf(x.x, y.x), base = mx == -INFINITY ? 0.f : mx;
    fx = exp2f(x.x - base);
    fy = exp2f(y.x - base);
    return make_float2(mx, x.y * fx + y.y * fy);
}

// Part i of a split that CTA c has the first part of lies in slot 2(c + i), the first in 2c + 1.
__device__ __forceinline__ int part_slot(int c, int i) { return 2 * (c + i) + (i == 0 ? 1 : 0); }

// Maximum and sum of a row from its parts, by a warp.
__device__ __forceinline__ float2 join_ml(const float2* part_ml, int R, int c, int parts, int r) {
    const int lane = threadIdx.x & 31;
    float2 x = make_float2(-INFINITY, 0.f);
    float f0, f1;
    for (int i = lane; i < parts; i += 32) x = join_two(x, part_ml[part_slot(c, i) * R + r], f0, f1);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        x = join_two(x, make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o)), f0, f1);
    return x;
}

// Second launch.  The last rows·ctas blocks: row j mod rows of the (sequence, head tile)
// whose first part CTA j / rows wrote, each group of E/4 threads taking some of the
// parts.  The `adders` blocks in front (with weights): weights[b][kv head][j] += Σ over the
// group of exp(s_j − maximum) / sum for a share of the slots; a split row's maximum and sum
// come from its parts again, so that both run at once.
template <typename T, int E, int R, int kUnit, int kExtra>
__global__ void __launch_bounds__(kThreads, 8) attention_join(AttnArgs a, int rows, int ctas, int adders) {
    constexpr int LE = E / 4;                             // lanes per row of 16-byte vectors
    constexpr int NP = kThreads / LE;                     // parts at once
    __shared__ __align__(16) union {
        struct {
            float acc[NP][E];
            float2 ml[NP];
        } j;
        struct {
            SplitShared split;
            int first[32], last[32];      // CTAs with the parts of a query head
            float2 row[32];               // its maximum, and 1 / its sum (0: no score)
        } w;
    } sh;
    const int t = threadIdx.x;
    if ((int)blockIdx.x >= adders) {
        wait_before();
        const int c = (blockIdx.x - adders) / rows, r = (blockIdx.x - adders) % rows;
        const int4 w = a.join[c];
        const int r0 = (w.y % a.tiles) * R;
        if (w.z == 0 || r0 + r >= a.group) return;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        float2 ml = make_float2(-INFINITY, 0.f);
        float f0, f1;
#pragma unroll 4
        for (int i = t / LE; i < w.z; i += NP) {
            const int slot = part_slot(c, i);
            const float4 y = *reinterpret_cast<const float4*>(a.part_acc + ((int64_t)slot * R + r) * E + (t % LE) * 4);
            ml = join_two(ml, a.part_ml[slot * R + r], f0, f1);
            x.x = x.x * f0 + y.x * f1;
            x.y = x.y * f0 + y.y * f1;
            x.z = x.z * f0 + y.z * f1;
            x.w = x.w * f0 + y.w * f1;
        }
        *reinterpret_cast<float4*>(&sh.j.acc[t / LE][(t % LE) * 4]) = x;
        if (t % LE == 0) sh.j.ml[t / LE] = ml;
        __syncthreads();
        if (t < E) {
            float sum = sh.j.acc[0][t];
            ml = sh.j.ml[0];
#pragma unroll
            for (int i = 1; i < NP; ++i) {
                ml = join_two(ml, sh.j.ml[i], f0, f1);
                sum = sum * f0 + sh.j.acc[i][t] * f1;
            }
            write_row<T, E>(a, w.x, (w.y / a.tiles) * a.group + r0 + r, t, sum, ml.x, ml.y);
        }
        return;
    }
    // The first launch's split again, which rests on the call's arguments alone, as do the
    // weights so far: all of it goes ahead of the wait for the first launch.
    const int heads = a.KH * a.tiles;
    Split s = split_begin<kUnit, kExtra>(a.c, a.B, heads, ctas, blockIdx.x, adders, sh.w.split);
    bool waited = false;
    while (const int c1 = s.segment()) {
        const int end = s.end_slot<kUnit>(c1);
        const int kvh = s.h / a.tiles;
        // a chunk's weights are added up by the block that has it for the first head tile
        if (s.h % a.tiles == 0) {
            const int64_t row0 = (int64_t)s.b * a.QH + kvh * a.group;
            float* w = a.weights + ((int64_t)s.b * a.KH + kvh) * a.c.slots;
            int held = -1;            // the heads from here have their rows in shared memory
            // four slots a thread at once: their loads do not wait for one another
            for (int j0 = s.first_slot<kUnit>(s.chunk) + t; j0 - t < end; j0 += 4 * kThreads) {
                float sum[4], add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = j0 + i * kThreads < end ? w[j0 + i * kThreads] : 0.f;
                for (int g0 = 0; g0 < a.group; g0 += 32) {
                    const int n = min(32, a.group - g0);
                    if (held != g0) {
                        held = g0;
                        __syncthreads();
                        if (t < n) {
                            // head tile h of sequence b has units before·heads + h·chunks + [0, chunks)
                            const long long u = s.before * heads + (long long)(s.h + (g0 + t) / R) * s.chunks;
                            sh.w.first[t] = s.owner(u + s.extra);
                            sh.w.last[t] = s.owner(u + s.chunks - 1);
                        }
                        if (!waited) wait_before();
                        waited = true;
                        __syncthreads();
                        for (int g = t / 32; g < n; g += kThreads / 32) {
                            const int first = sh.w.first[g], parts = sh.w.last[g] - first + 1;
                            const float2 x = parts == 1 ? a.row_ml[row0 + g0 + g]
                                                        : join_ml(a.part_ml, R, first, parts, (g0 + g) % R);
                            if (t % 32 == 0)
                                sh.w.row[g] = x.y == 0.f ? make_float2(0.f, 0.f) : make_float2(x.x, 1.f / x.y);
                        }
                        __syncthreads();
                    }
                    for (int g = 0; g < n; ++g) {
                        const float2 x = sh.w.row[g];
                        const float* sc = a.scores + (row0 + g0 + g) * a.c.slots;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (j0 + i * kThreads < end)
                                add[i] = fmaf(exp2f(fmaf(sc[j0 + i * kThreads], a.scale2, -x.x)), x.y, add[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = j0 + i * kThreads;
                    if (j >= end) continue;
                    // a row that is not finite gives its slots NaN, but none to those without a page
                    if (add[i] != add[i] && a.c.offset(a.c.table + (int64_t)s.b * a.c.max_pages, j) < 0) add[i] = 0.f;
                    if (add[i] != 0.f) w[j] = sum[i] + add[i];
                }
            }
        }
        split_next<kUnit>(s, c1, a.c, heads);
    }
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// Query heads that one pass over the keys serves.
int rows_per_tile(int64_t group, int dtype) {
    if (dtype != NNOP_F32) return group <= 8 ? 8 : group <= 16 ? 16 : 32;
    return group <= 1 ? 1 : group <= 2 ? 2 : group <= 4 ? 4 : 8;
}

struct Layout {
    size_t join, ml, acc, scores, rows, bytes;
};
Layout layout(int64_t E, int64_t QH, int64_t KH, int64_t B, int64_t slots, bool weights, int dtype) {
    const size_t R = rows_per_tile(QH / KH, dtype);
    Layout w;
    w.join = 0;
    w.ml = align256(sizeof(int4) * kMaxCtas);
    w.acc = w.ml + align256(sizeof(float2) * 2 * kMaxCtas * R);
    w.scores = w.acc + align256(sizeof(float) * 2 * kMaxCtas * R * E);
    w.rows = w.scores + (weights ? align256(sizeof(float) * (size_t)B * QH * slots) : 0);
    w.bytes = w.rows + (weights ? align256(sizeof(float2) * (size_t)B * QH) : 0);
    return w;
}

int check_heads(int64_t E, int64_t QH, int64_t KH, int64_t B) {
    if (E <= 0 || QH <= 0 || KH <= 0 || B < 0) return fail(NNOP_ERR_SHAPE, "paged_attention: invalid dimensions");
    if (QH % KH != 0)
        return fail(NNOP_ERR_SHAPE, "Number of query heads `" + std::to_string(QH) +
                                        "` must be divisible by number of KV heads `" + std::to_string(KH) + "`.");
    if (QH > 65535) return fail(NNOP_ERR_SHAPE, "paged_attention: too many heads");
    return NNOP_OK;
}

template <typename T, int E, int R>
int launch(const AttnArgs& a, cudaStream_t s) {
    int G;
    constexpr bool f32 = std::is_same<T, float>::value;
    if constexpr (f32) {
        G = std::min(kMaxCtas, 3 * num_sms());
        attention_simt<E, R><<<G, kThreads, 0, s>>>(a);
    } else {
        constexpr int NT = R == 8 ? 1 : 2, WT = R / (8 * NT);
        G = std::min(kMaxCtas, mma_ctas(NT) * num_sms());
        if (a.c.page_size.d % 16 == 0)
            attention_mma<T, E, NT, WT, true><<<G, kThreads, 0, s>>>(a);
        else
            attention_mma<T, E, NT, WT, false><<<G, kThreads, 0, s>>>(a);
    }
    if (const int rc = check_launch("paged_attention")) return rc;
    const int rows = std::min(R, a.group), adders = a.weights != nullptr ? 8 * num_sms() : 0;
    return launch_dependent("paged_attention",
                            attention_join<T, E, R, f32 ? SimtShape<E>::kUnit : MmaShape<E>::kUnit,
                                           f32 ? kSimtExtra : mma_extra(R == 8 ? 1 : 2)>,
                            dim3(adders + G * rows), dim3(kThreads), 0, s, a, rows, G, adders);
}

template <typename T, int E>
int launch_rows(const AttnArgs& a, int rows, cudaStream_t s) {
    if constexpr (std::is_same<T, float>::value) {
        switch (rows) {
            case 1: return launch<T, E, 1>(a, s);
            case 2: return launch<T, E, 2>(a, s);
            case 4: return launch<T, E, 4>(a, s);
            default: return launch<T, E, 8>(a, s);
        }
    } else {
        switch (rows) {
            case 8: return launch<T, E, 8>(a, s);
            case 16: return launch<T, E, 16>(a, s);
            default: return launch<T, E, 32>(a, s);
        }
    }
}

}  // namespace
}  // namespace paged
}  // namespace nnop

using namespace nnop;

extern "C" {

size_t nnop_paged_attention_fwd_workspace_size(int64_t E, int64_t QH, int64_t KH, int64_t B, int64_t page_size,
                                               int64_t max_pages, int has_weights, int dtype) {
    if (E <= 0 || QH <= 0 || KH <= 0 || B <= 0 || page_size <= 0 || max_pages < 0) return 0;
    return paged::layout(E, QH, KH, B, page_size * max_pages, has_weights != 0, dtype).bytes;
}

int nnop_paged_attention_fwd(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                             const int32_t* lengths, float* weights, void* o, float* lse, void* workspace,
                             size_t workspace_bytes, int64_t E, int64_t QH, int64_t KH, int64_t B, int64_t pages,
                             int64_t page_size, int64_t max_pages, int64_t page_stride, int64_t head_stride,
                             int64_t row_stride, int dtype, void* stream) {
    return paged::guarded("paged_attention", [&]() -> int {
        paged::AttnArgs a{};
        if (const int rc = paged::check_heads(E, QH, KH, B)) return rc;
        if (const int rc = paged::check_cache("paged_attention", a.c, block_table, lengths, E, KH, B, pages, page_size,
                                              max_pages, page_stride, head_stride, row_stride, dtype))
            return rc;
        if (B == 0) return NNOP_OK;
        // the split's unit numbers times its CTAs stay within 64 bits
        if ((double)B * (double)QH * (a.c.slots / 16 + 32) > 9e15)
            return fail(NNOP_ERR_SHAPE, "paged_attention: too many slots in all");
        if (!q || !o || !lse || !workspace || (pages > 0 && (!k_cache || !v_cache)))
            return fail(NNOP_ERR_ARG, "paged_attention: NULL pointer");
        if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(o))
            return fail(NNOP_ERR_ALIGN, "paged_attention: tensors must be 16-byte aligned");
        const paged::Layout w = paged::layout(E, QH, KH, B, a.c.slots, weights != nullptr, dtype);
        if (workspace_bytes < w.bytes)
            return fail(NNOP_ERR_WORKSPACE, "paged_attention: workspace too small (" +
                                                std::to_string(workspace_bytes) + " < " + std::to_string(w.bytes) + ")");
        if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
            return fail(NNOP_ERR_ALIGN, "paged_attention: workspace must be 256-byte aligned");
        a.q = q;
        a.k = k_cache;
        a.v = v_cache;
        a.o = o;
        a.lse = lse;
        a.weights = weights;
        a.B = B;
        a.QH = (int)QH;
        a.KH = (int)KH;
        a.group = (int)(QH / KH);
        const int R = paged::rows_per_tile(a.group, dtype);
        a.tiles = (a.group + R - 1) / R;
        char* base = static_cast<char*>(workspace);
        a.join = reinterpret_cast<int4*>(base + w.join);
        a.part_ml = reinterpret_cast<float2*>(base + w.ml);
        a.part_acc = reinterpret_cast<float*>(base + w.acc);
        a.scores = weights ? reinterpret_cast<float*>(base + w.scores) : nullptr;
        a.row_ml = weights ? reinterpret_cast<float2*>(base + w.rows) : nullptr;
        const cudaStream_t s = (cudaStream_t)stream;
        const float sc = (float)(1.0 / std::sqrt((double)E));
        // scale rounded to the dtype, as flash_attention has it
        a.scale2 = paged::kLog2e * (dtype == NNOP_BF16 ? __bfloat162float(__float2bfloat16_rn(sc))
                                    : dtype == NNOP_F16 ? __half2float(__float2half_rn(sc)) : sc);
        NNOP_DISPATCH_DTYPE(dtype, T, {
            switch (E) {
                case 16: return paged::launch_rows<T, 16>(a, R, s);
                case 32: return paged::launch_rows<T, 32>(a, R, s);
                case 64: return paged::launch_rows<T, 64>(a, R, s);
                default: return paged::launch_rows<T, 128>(a, R, s);
            }
        });
        return NNOP_OK;
    });
}

}  // extern "C"
