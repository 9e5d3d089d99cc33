// moe_layer.cu — a whole mixture-of-experts layer for a few tokens.
//
// For every route r = (token t, slot k) with expert e = topk_ids[t][k]:
//   xq, rs1 = smoothquant(x[t], smooth1[e])
//   [g | u] = float(w13[e] xq) * (rs1 * s13[e])
//   h       = g / (1 + exp(-g)) * u * smooth2[e];  hq, rs2 = its quantisation
//   d       = float(w2[e] hq) * (rs2 * s2[e])
//   out[t]  = sum over k of topk_w[t][k] * d, in slot order
// A route whose id is outside [0, experts) adds nothing.  A NaN or an infinity
// among xs or h makes the token's whole output NaN (smoothquant by itself would
// drop it from the maximum and go on with a wrong row).
//
// What bounds it is reading the weights of the experts that were chosen, once.
// Blocks of an expert's routes (up to 8 NT of them) meet its weight rows in
// tiles of 16 rows; every block of the grid (one an SM) takes an equal run of
// the tiles, which lie one after another in memory, and each of its eight warps
// an equal run of their 128-byte pieces.  Weights stream through a ring of
// cp.async stages of the warp's own, so that no barrier stands between loading
// and multiplying; the routes' int8 rows lie in shared memory.
// mma.m16n8k32: weight rows are the 16, routes the 8 columns.  A warp has most
// tiles to itself and ends them in registers; the tiles between two warps' runs
// meet in shared memory by integer adds.  (Eight warps on every tile, an eighth
// of its columns each, add and wait 16 times as often: 64 tokens, 8 experts,
// 2 slots, 4096 x 14336: 337 us, 295 this way; 58 tokens, 128 experts, 3 slots,
// 4832 x 336: 102 and 76; but 16 tokens, where few sums wait and each weight row
// is read in longer pieces, 222 and 227.)
//
// 1 token, 8 experts, 2 slots, 4096 x 14336: 64 us (353 MB: 5.5 TB/s of the 6.6
// that a copy moves); 16 tokens: 227 us (6.2); 24 tokens, 32 experts, 5 slots,
// 4096 x 1456: 94 us (6.0).
//
//   moe_quant_x_kernel  smoothquant of each route's token; clears what the others add to
//   moe_up_kernel       gate and up rows (8 + 8 a tile, so one thread has both), SwiGLU;
//                       leaves h in fp32 and the largest |h| of each route
//   moe_quant_h_kernel  h to int8
//   moe_down_kernel     w2; slices of the inner dimension are added as integers
//                       (exact, in any order)
//   moe_sum_kernel      scales, weighs and adds the slots
// The two products start to stream their weights before the kernel in front of
// them is done (programmatic launch).  Quantising once in small kernels beats
// doing it in the products, where every block repeats it for its experts behind
// its own weight loads (16 tokens: 8 to 13 us a time; 4 us this way).
#include "common.cuh"
#include "kernels.h"
#include "sq_math.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2sq {

namespace {

constexpr uint32_t kWarps = 8;
constexpr uint32_t kThreads = kWarps * 32;
constexpr uint32_t kTile = 2048;         // bytes of a warp's stage: 16 rows of 128
constexpr uint32_t kSliceMost = 4096;    // inner elements of h that a block of the second kernel holds at a time
constexpr uint32_t kSmemMost = 231424;   // dynamic shared memory: 227 KB, less 1 KB for what is static

struct Lists {
    uint16_t *first, *block, *order;  // [E + 1] first route and first block of an expert, [R] routes by expert
};

struct Params {
    MoeLayer m;
    int8_t *xq, *hq;  // [R][hidden], [R][inter]
    float* rs1;       // [R]
    uint32_t* top;    // [R] largest |h|, as bits
    float* h;         // [R][inter]
    int32_t* acc;     // [R][hidden]
    uint32_t slices, slice;  // of the second kernel: slices of `slice` inner elements
};

// Shared memory of both products: the ring, the routes' rows, the sums, the lists.
template <int NT, int STAGES>
struct Smem {
    static constexpr uint32_t ring = kWarps * STAGES * kTile;
    static constexpr uint32_t pitch = NT == 1 ? 8 : NT == 2 ? 24 : 36;  // ints of a row of sums: two-way bank conflicts at most
    static constexpr uint32_t tile_sums = 16 * pitch;
    static constexpr uint32_t sums = (kWarps - 1) * tile_sums * 4;      // of the tiles between two warps' runs
    __host__ __device__ static constexpr uint32_t row_pitch(uint32_t k) { return (k + 127) / 128 * 128 + 16; }
    __host__ __device__ static constexpr uint32_t rows(uint32_t k) { return 8 * NT * row_pitch(k); }
    __host__ __device__ static constexpr uint32_t lists(uint32_t experts, uint32_t routes)
    {
        return (2 * (experts + 1) + routes) * 2;
    }
    static constexpr uint64_t total(uint32_t k, uint32_t experts, uint32_t routes)
    {
        return (uint64_t)ring + rows(k) + sums + lists(experts, routes);
    }
};

// (256 bytes a trip to memory: with 128, 24 tokens over 32 experts took 99 us, with 256 they take 94)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes)
{
    asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ float2 pair_to_f2(uint32_t w);
template <>
__device__ __forceinline__ float2 pair_to_f2<__half>(uint32_t w)
{
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 pair_to_f2<__nv_bfloat16>(uint32_t w)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Eight activations times their smooth scales, in fp32 (smoothquant's first step).
template <typename T>
__device__ __forceinline__ void smoothed(const uint4& w, const float4& s0, const float4& s1, float (&f)[8])
{
    const float2 a = pair_to_f2<T>(w.x), b = pair_to_f2<T>(w.y), c = pair_to_f2<T>(w.z), d = pair_to_f2<T>(w.w);
    f[0] = __fmul_rn(a.x, s0.x), f[1] = __fmul_rn(a.y, s0.y), f[2] = __fmul_rn(b.x, s0.z), f[3] = __fmul_rn(b.y, s0.w);
    f[4] = __fmul_rn(c.x, s1.x), f[5] = __fmul_rn(c.y, s1.y), f[6] = __fmul_rn(d.x, s1.z), f[7] = __fmul_rn(d.y, s1.w);
}

// The low byte of quant1's result; integral qmax takes the form without conversions.
__device__ __forceinline__ uint32_t quant_byte(float xs, float inv, float qmax, bool whole)
{
    return whole ? quant_bits(xs, inv, qmax) : (uint32_t)(uint8_t)quant1(xs, inv, qmax);
}
__device__ __forceinline__ uint32_t quant4(float a, float b, float c, float d, float inv, float qmax, bool whole)
{
    return pack_low_bytes(quant_byte(a, inv, qmax, whole), quant_byte(b, inv, qmax, whole), quant_byte(c, inv, qmax, whole),
                          quant_byte(d, inv, qmax, whole));
}

// The scale of a row whose largest magnitude has these bits.  Magnitudes are compared as integers, which order as the
// floats do with a NaN above infinity: a row that holds either has a NaN for its scale, and so for everything after it.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ float scale_of(uint32_t top, float qmax)
{
    return top < 0x7f800000u ? row_scale_of(__uint_as_float(top), qmax) : __uint_as_float(0x7fffffffu);
}

// A block a route: hidden <= 16384 is at most 64 values a thread, read once.
template <typename T>
__global__ void __launch_bounds__(kThreads) moe_quant_x_kernel(Params p)
{
    __shared__ uint32_t warp_max[kWarps];
    griddep_wait();
    griddep_launch_dependents();
    const MoeLayer& m = p.m;
    const uint32_t r = blockIdx.x, tid = threadIdx.x, H = m.hidden;
    const uint32_t e = (uint32_t)__ldg(m.topk_ids + r);
    const T* x = static_cast<const T*>(m.x) + (uint64_t)(r / m.topk) * m.x_stride;
    uint4 xw[8];
    float4 sw[8][2];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t k = (i * kThreads + tid) * 8;
        xw[i] = k < H ? __ldg(reinterpret_cast<const uint4*>(x + k)) : make_uint4(0, 0, 0, 0);
    }
    if (tid == 0) p.top[r] = 0;
    if (e >= m.experts) return;
    const float* sm = m.smooth1 + (uint64_t)e * H;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t k = (i * kThreads + tid) * 8;
        sw[i][0] = sw[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k < H) {
            sw[i][0] = __ldg(reinterpret_cast<const float4*>(sm + k));
            sw[i][1] = __ldg(reinterpret_cast<const float4*>(sm + k) + 1);
        }
    }
    if (p.slices > 1)  // the down product adds its slices up from zero
        for (uint32_t i = tid; i < H / 4; i += kThreads) reinterpret_cast<int4*>(p.acc + (uint64_t)r * H)[i] = make_int4(0, 0, 0, 0);
    float f[8][8];
    uint32_t mx = 0;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        smoothed<T>(xw[i], sw[i][0], sw[i][1], f[i]);
#pragma unroll
        for (int c = 0; c < 8; ++c) mx = max(mx, magnitude(f[i][c]));
    }
    mx = __reduce_max_sync(0xffffffffu, mx);
    if ((tid & 31) == 0) warp_max[tid / 32] = mx;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) mx = max(mx, warp_max[w]);
    const float rs = scale_of(mx, m.qmax), inv = inv_scale_of(rs);
    const bool whole = m.qmax == rintf(m.qmax);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t k = (i * kThreads + tid) * 8;
        if (k < H)
            *reinterpret_cast<uint2*>(p.xq + (uint64_t)r * H + k) =
                make_uint2(quant4(f[i][0], f[i][1], f[i][2], f[i][3], inv, m.qmax, whole),
                           quant4(f[i][4], f[i][5], f[i][6], f[i][7], inv, m.qmax, whole));
    }
    if (tid == 0) p.rs1[r] = rs;
}

// grid (pieces of 2048, routes)
__global__ void __launch_bounds__(kThreads) moe_quant_h_kernel(Params p)
{
    // (the down product behind this kernel may start once the up product has: it touches only the layer's inputs
    // until this kernel, which waits for the up product, is done)
    griddep_launch_dependents();
    const MoeLayer& m = p.m;
    const uint32_t r = blockIdx.y, k = (blockIdx.x * kThreads + threadIdx.x) * 8;
    const bool there = (uint32_t)__ldg(m.topk_ids + r) < m.experts && k < m.inter;
    griddep_wait();
    if (!there) return;
    const float4* h = reinterpret_cast<const float4*>(p.h + (uint64_t)r * m.inter + k);
    const float4 a = h[0], b = h[1];
    const float inv = inv_scale_of(scale_of(p.top[r], m.qmax));
    const bool whole = m.qmax == rintf(m.qmax);
    *reinterpret_cast<uint2*>(p.hq + (uint64_t)r * m.inter + k) =
        make_uint2(quant4(a.x, a.y, a.z, a.w, inv, m.qmax, whole), quant4(b.x, b.y, b.z, b.w, inv, m.qmax, whole));
}

// Routes grouped by expert, in their own order, and blocks of at most `most`
// routes; every block of both kernels computes the same lists.  `scratch`:
// [R] uint16 and [E] uint32 of shared memory that is free until the next barrier.
__device__ __forceinline__ void make_lists(const MoeLayer& m, uint32_t most, const Lists& l, uint32_t* scratch)
{
    __shared__ uint32_t warp_rows[kWarps], warp_blocks[kWarps];
    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31, routes = m.tokens * m.topk;
    uint32_t* count = scratch;
    uint16_t* rank = reinterpret_cast<uint16_t*>(scratch + m.experts);
    for (uint32_t e = tid; e < m.experts; e += kThreads) count[e] = 0;
    // the ranks' places hold the experts first: one trip to memory for all of them
    for (uint32_t r = tid; r < routes; r += kThreads)
        rank[r] = (uint16_t)min((uint32_t)__ldg(m.topk_ids + r), m.experts);
    __syncthreads();
    if (warp == 0)
        for (uint32_t base = 0; base < routes; base += 32) {
            const uint32_t r = base + lane;
            const uint32_t e = r < routes ? rank[r] : m.experts;
            const bool valid = e < m.experts;
            const uint32_t same = __match_any_sync(0xffffffffu, e);
            const uint32_t before = valid ? count[e] : 0;
            __syncwarp();
            if (valid) {
                rank[r] = (uint16_t)(before + __popc(same & ((1u << lane) - 1)));
                if (lane == __ffs(same) - 1) count[e] = before + __popc(same);
            }
            __syncwarp();
        }
    __syncthreads();
    uint32_t row0 = 0, block0 = 0;
    for (uint32_t base = 0; base < m.experts; base += kThreads) {
        const uint32_t e = base + tid;
        const uint32_t n = e < m.experts ? count[e] : 0, b = (n + most - 1) / most;
        uint32_t ni = n, bi = b;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, ni, off), y = __shfl_up_sync(0xffffffffu, bi, off);
            if (lane >= (uint32_t)off) {
                ni += x;
                bi += y;
            }
        }
        if (lane == 31) {
            warp_rows[warp] = ni;
            warp_blocks[warp] = bi;
        }
        __syncthreads();
        uint32_t rb = row0, bb = block0;
        for (uint32_t w = 0; w < kWarps; ++w) {
            if (w < warp) {
                rb += warp_rows[w];
                bb += warp_blocks[w];
            }
            row0 += warp_rows[w];
            block0 += warp_blocks[w];
        }
        if (e < m.experts) {
            l.first[e] = (uint16_t)(rb + ni - n);
            l.block[e] = (uint16_t)(bb + bi - b);
        }
        __syncthreads();
    }
    if (tid == 0) {
        l.first[m.experts] = (uint16_t)row0;
        l.block[m.experts] = (uint16_t)block0;
    }
    for (uint32_t r = tid; r < routes; r += kThreads) {
        const uint32_t e = (uint32_t)__ldg(m.topk_ids + r);
        if (e < m.experts) l.order[l.first[e] + rank[r]] = (uint16_t)r;
    }
    __syncthreads();
}

// The expert that block `b` belongs to.
__device__ __forceinline__ uint32_t expert_of(const Lists& l, uint32_t experts, uint32_t b)
{
    uint32_t lo = 0, hi = experts;  // the last expert that starts at or before b
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (l.block[mid] <= b)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

struct Block {
    uint32_t expert, r0, count;  // routes order[r0 .. r0 + count)
};
template <int NT>
__device__ __forceinline__ Block block_at(const Lists& l, uint32_t experts, uint32_t b)
{
    Block k;
    k.expert = expert_of(l, experts, b);
    k.r0 = l.first[k.expert] + (b - l.block[k.expert]) * 8 * NT;
    k.count = min(8u * NT, (uint32_t)l.first[k.expert + 1] - k.r0);
    return k;
}

// Equal runs of `total` units for `blocks` blocks: the first `rest` get one more.
struct Split {
    uint32_t each, rest;
    __device__ __forceinline__ Split(uint32_t total, uint32_t blocks) : each(total / blocks), rest(total % blocks) {}
    __device__ __forceinline__ uint32_t begin(uint32_t i) const { return i * each + min(i, rest); }
};

// The block's int8 rows (bytes k0 .. k0 + depth of rows of `width`) on their way into shared memory: the first
// FLY x 16 bytes of each thread can be fetched early and stored when the rows before them are no longer read.
struct RowCopy {
    static constexpr uint32_t FLY = 8;
    uint4 v[FLY];
    template <typename F>
    __device__ __forceinline__ void each(uint32_t i0, uint32_t depth, uint32_t count, F&& f)
    {
        const uint32_t chunks = depth / 16, all = count * chunks;
#pragma unroll
        for (uint32_t n = 0; n < FLY; ++n) {
            const uint32_t i = i0 + n * kThreads, t = i / chunks;
            if (i < all) f(v[n], t, (i - t * chunks) * 16);
        }
    }
    __device__ __forceinline__ void fetch(uint32_t i0, const int8_t* src, uint64_t width, uint32_t k0, uint32_t depth,
                                          const uint16_t* order, uint32_t count)
    {
        each(i0, depth, count, [&](uint4& x, uint32_t t, uint32_t k) {
            x = *reinterpret_cast<const uint4*>(src + order[t] * width + k0 + k);
        });
    }
    // stores what was fetched from i0 = threadIdx.x on, then fetches and stores the rest
    __device__ __forceinline__ void finish(uint8_t* rows, uint32_t row_pitch, const int8_t* src, uint64_t width, uint32_t k0,
                                           uint32_t depth, const uint16_t* order, uint32_t count)
    {
        for (uint32_t i0 = threadIdx.x;;) {
            each(i0, depth, count, [&](uint4& x, uint32_t t, uint32_t k) {
                *reinterpret_cast<uint4*>(rows + t * row_pitch + k) = x;
            });
            i0 += FLY * kThreads;
            if (i0 - threadIdx.x >= count * (depth / 16)) break;
            fetch(i0, src, width, k0, depth, order, count);
        }
    }
};

// The pieces of a block's row tiles, one tile's 128-byte pieces after another's, in equal runs for the warps.
struct Runs {
    uint32_t total, pieces;
    __device__ __forceinline__ Runs(uint32_t tiles, uint32_t pieces_) : total(tiles * pieces_), pieces(pieces_) {}
    __device__ __forceinline__ uint32_t begin(uint32_t w) const
    {
        return total / kWarps * w + total % kWarps * w / kWarps;
    }
    // Warp w's run begins inside a tile, and is the first to: that tile (its sums meet in place w - 1), else ~0.
    __device__ __forceinline__ uint32_t cut_tile(uint32_t w) const
    {
        if (w == 0) return ~0u;
        const uint32_t q = begin(w), t = q / pieces;
        return q == t * pieces || begin(w - 1) > t * pieces ? ~0u : t;
    }
    // The place of a cut tile's sums, for a warp whose run begins in it or before it.
    __device__ __forceinline__ uint32_t place_of(uint32_t w, uint32_t t) const
    {
        if (begin(w) <= t * pieces) ++w;
        while (w > 1 && begin(w - 1) > t * pieces) --w;
        return w - 1;
    }
};

// int32 products of a tile's 16 weight rows with the block's routes, over `count` of its pieces from p0 on.
template <int NT, int STAGES, typename Next>
__device__ __forceinline__ void tile_product(uint32_t p0, uint32_t count, uint32_t live, uint32_t ring_base,
                                             uint32_t rows_base, uint32_t row_pitch, uint32_t& slot, int (&acc)[NT][4],
                                             Next&& next)
{
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t arow = (lane & 7) + ((lane >> 3) & 1) * 8, asel = lane >> 4;
    uint32_t brow = rows_base + (lane & 7) * row_pitch + (lane >> 3) * 16 + p0 * 128;
    int odd[NT][4];  // a second chain of products: one waits half as long for its own
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][i] = odd[nt][i] = 0;
#pragma unroll 1
    for (uint32_t n = 0; n < count; ++n, brow += 128) {
        cp_async_wait<STAGES - 2>();
        __syncwarp();
        // the slot that the last step freed takes the piece STAGES - 1 steps ahead
        next();
        const uint32_t a_at = ring_base + slot * kTile + arow * 128;
        if (++slot == STAGES) slot = 0;
        uint32_t a[4][4];
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q) ldsm4(a_at + (((q * 2 + asel) ^ (arow & 7)) * 16), a[q]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            if (nt == 0 || nt < live) {
                const uint32_t b_at = brow + nt * 8 * row_pitch;
                uint32_t b[2][4];
                ldsm4(b_at, b[0]);
                ldsm4(b_at + 64, b[1]);
                mma_s8(acc[nt], a[0], b[0][0], b[0][1]);
                mma_s8(odd[nt], a[1], b[0][2], b[0][3]);
                mma_s8(acc[nt], a[2], b[1][0], b[1][1]);
                mma_s8(odd[nt], a[3], b[1][2], b[1][3]);
            }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][i] += odd[nt][i];
}

// Adds a warp's products into a cut tile's sums in shared memory (zero before), and takes them out again.
template <int NT, uint32_t PITCH>
__device__ __forceinline__ void add_sums(int* sums, const int (&acc)[NT][4], uint32_t live)
{
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, tig = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
        if (nt == 0 || nt < live)
#pragma unroll
            for (int i = 0; i < 4; ++i) atomicAdd(sums + (g + i / 2 * 8) * PITCH + nt * 8 + 2 * tig + (i & 1), acc[nt][i]);
}
template <int NT, uint32_t PITCH>
__device__ __forceinline__ void take_sums(int* sums, int (&acc)[NT][4])
{
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, tig = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int* at = sums + (g + i / 2 * 8) * PITCH + nt * 8 + 2 * tig + (i & 1);
            acc[nt][i] = *at;
            *at = 0;
        }
}

// Gate and up rows.  Row tiles: block of routes x 8 inner elements.
template <int NT, int STAGES>
__global__ void __launch_bounds__(kThreads, 1) moe_up_kernel(Params p)
{
    using S = Smem<NT, STAGES>;
    extern __shared__ __align__(128) uint8_t moe_smem[];
    __shared__ float rs1[8 * NT];
    __shared__ uint32_t top[8 * NT];
    const MoeLayer& m = p.m;
    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const uint32_t H = m.hidden, I = m.inter;
    const uint32_t row_pitch = S::row_pitch(H);
    uint8_t* rows = moe_smem + S::ring;
    int* sums = reinterpret_cast<int*>(rows + S::rows(H));
    uint16_t* list = reinterpret_cast<uint16_t*>(reinterpret_cast<uint8_t*>(sums) + S::sums);
    const Lists l{list, list + m.experts + 1, list + 2 * (m.experts + 1)};

    // before the wait: only what the layer's inputs say (the first kernel has waited for them)
    make_lists(m, 8 * NT, l, reinterpret_cast<uint32_t*>(moe_smem));
    for (uint32_t i = tid; i < S::sums / 4; i += kThreads) sums[i] = 0;

    const uint32_t per_block = I / 8, total = l.block[m.experts] * per_block;
    const Split split(total, gridDim.x);
    const uint32_t begin = split.begin(blockIdx.x), end = split.begin(blockIdx.x + 1);

    // producer: this warp's next piece pq of its run in the units pu .. pu + pn of one block of routes, and its address
    const uint32_t pieces = (H + 127) / 128;
    const uint32_t ring_base = smem_u32(moe_smem) + warp * STAGES * kTile;
    const uint32_t lrow = lane / 8, lchunk = lane & 7;
    uint32_t pu = begin, pn = 0, pq = 0, pend = 0, pp = 0, pslot = 0;
    const int8_t* src = nullptr;
    auto settle = [&]() {  // on to the next run that is not empty
        while (pq == pend && (pu += pn) < end) {
            const uint32_t pb = pu / per_block, pj = pu - pb * per_block;
            pn = min(per_block - pj, end - pu);
            const Runs runs(pn, pieces);
            pq = runs.begin(warp);
            pend = runs.begin(warp + 1);
            const uint32_t t = pq / pieces;
            pp = pq - t * pieces;
            src = m.w13 + ((uint64_t)expert_of(l, m.experts, pb) * 2 * I + (pj + t) * 8 + lrow) * H + lchunk * 16;
        }
    };
    auto load = [&]() {
        if (pq < pend) {
            const uint32_t at = pp * 128 + lchunk * 16;
            const uint32_t bytes = at < H ? 16u : 0u;
            const uint32_t dst = ring_base + pslot * kTile;
            const int8_t* s = src + pp * 128;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t r = i * 4 + lrow;  // 0..7 gate, 8..15 up
                const int8_t* row = s + (uint64_t)((i & 1) * 4 + (i >> 1) * I) * H;
                // (the last piece may reach past the row: nothing is read there)
                cp_async16(dst + r * 128 + ((lchunk ^ (r & 7)) * 16), bytes ? row : m.w13, bytes);
            }
            if (++pp == pieces) {
                pp = 0;
                src += (uint64_t)8 * H;
            }
            if (++pq == pend) settle();
        }
        cp_async_commit();
        if (++pslot == STAGES) pslot = 0;
    };
    if (begin < end) {
        settle();
#pragma unroll 1
        for (int i = 0; i < STAGES - 1; ++i) load();
    }
    griddep_wait();
    griddep_launch_dependents();
    if (begin == end) return;

    uint32_t slot = 0;
    uint32_t b = begin / per_block, j = begin % per_block;
    RowCopy copy;
    Block cur = block_at<NT>(l, m.experts, b);
    copy.fetch(tid, p.xq, H, 0, H, l.order + cur.r0, cur.count);
    const uint32_t g = lane >> 2, tig = lane & 3;
    for (uint32_t u = begin; u < end;) {
        const uint32_t e = cur.expert, r0 = cur.r0, count = cur.count;
        copy.finish(rows, row_pitch, p.xq, H, 0, H, l.order + r0, count);
        if (tid < count) {
            rs1[tid] = p.rs1[l.order[r0 + tid]];
            top[tid] = 0;
        }
        __syncthreads();
        const uint32_t live = (count + 7) / 8, here = min(per_block - j, end - u);
        if (u + here < end) {  // the next block's rows, behind this one's products
            cur = block_at<NT>(l, m.experts, b + 1);
            copy.fetch(tid, p.xq, H, 0, H, l.order + cur.r0, cur.count);
        }
        uint32_t mx[NT][2] = {};
        struct Scales {
            float gate, up, smooth;
        };
        auto scales = [&](uint32_t t) {  // of the thread's inner element of tile t
            const uint32_t at = (j + t) * 8 + g;
            const float* s = m.s13 + (uint64_t)e * 2 * I + at;
            return Scales{__ldg(s), __ldg(s + I), __ldg(m.smooth2 + (uint64_t)e * I + at)};
        };
        auto finish = [&](uint32_t t, const int (&acc)[NT][4], const Scales& s) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t tok = nt * 8 + 2 * tig + c;
                    if (tok >= count) continue;
                    const float gv = __fmul_rn((float)acc[nt][c], __fmul_rn(rs1[tok], s.gate));
                    const float uv = __fmul_rn((float)acc[nt][2 + c], __fmul_rn(rs1[tok], s.up));
                    const float hv = gv / (1.f + expf(-gv)) * uv * s.smooth;
                    p.h[(uint64_t)l.order[r0 + tok] * I + (j + t) * 8 + g] = hv;
                    mx[nt][c] = max(mx[nt][c], magnitude(hv));
                }
        };
        const Runs runs(here, pieces);
        uint32_t q = runs.begin(warp), t = q / pieces, p0 = q - t * pieces;
        const uint32_t qe = runs.begin(warp + 1);
        Scales sc = q < qe ? scales(t) : Scales{};
        int acc[NT][4];
        while (q < qe) {
            const uint32_t n = min(pieces - p0, qe - q);
            const Scales ahead = q + n < qe ? scales(t + 1) : Scales{};
            tile_product<NT, STAGES>(p0, n, live, ring_base, smem_u32(rows), row_pitch, slot, acc, load);
            if (n == pieces)
                finish(t, acc, sc);
            else
                add_sums<NT, S::pitch>(sums + runs.place_of(warp, t) * S::tile_sums, acc, live);
            sc = ahead;
            q += n;
            p0 = 0;
            ++t;
        }
        // the tiles between two runs, a warp each
        const uint32_t cut = runs.cut_tile(warp);
        if (cut != ~0u) sc = scales(cut);
        __syncthreads();
        if (cut != ~0u) {
            take_sums<NT, S::pitch>(sums + (warp - 1) * S::tile_sums, acc);
            finish(cut, acc, sc);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) mx[nt][c] = max(mx[nt][c], __shfl_xor_sync(0xffffffffu, mx[nt][c], off));
                const uint32_t tok = nt * 8 + 2 * tig + c;
                if (g == 0 && tok < count) atomicMax(top + tok, mx[nt][c]);
            }
        __syncthreads();  // (and the rows are read, and the sums are zero)
        if (tid < count) atomicMax(p.top + l.order[r0 + tid], top[tid]);
        u += here;
        ++b;
        j = 0;
    }
    cp_async_wait<0>();
}

// Down rows.  Row tiles: (block of routes, slice of the inner dimension) x 16 rows.
template <int NT, int STAGES>
__global__ void __launch_bounds__(kThreads, 1) moe_down_kernel(Params p)
{
    using S = Smem<NT, STAGES>;
    extern __shared__ __align__(128) uint8_t moe_smem[];
    const MoeLayer& m = p.m;
    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const uint32_t H = m.hidden, I = m.inter;
    const uint32_t row_pitch = S::row_pitch(p.slice);
    uint8_t* rows = moe_smem + S::ring;
    int* sums = reinterpret_cast<int*>(rows + S::rows(p.slice));
    uint16_t* list = reinterpret_cast<uint16_t*>(reinterpret_cast<uint8_t*>(sums) + S::sums);
    const Lists l{list, list + m.experts + 1, list + 2 * (m.experts + 1)};

    // before the wait: only what the layer's inputs say (the first kernel has waited for them)
    make_lists(m, 8 * NT, l, reinterpret_cast<uint32_t*>(moe_smem));
    for (uint32_t i = tid; i < S::sums / 4; i += kThreads) sums[i] = 0;
    const uint32_t per_slice = H / 16, per_block = per_slice * p.slices;
    const uint32_t total = l.block[m.experts] * per_block;
    const Split split(total, gridDim.x);
    const uint32_t begin = split.begin(blockIdx.x), end = split.begin(blockIdx.x + 1);

    const uint32_t ring_base = smem_u32(moe_smem) + warp * STAGES * kTile;
    const uint32_t lrow = lane / 8, lchunk = lane & 7;
    uint32_t pu = begin, pn = 0, pq = 0, pend = 0, pp = 0, ppieces = 0, pslot = 0;
    uint32_t left = 0;  // inner elements of the producer's slice
    const int8_t* src = nullptr;
    auto settle = [&]() {
        while (pq == pend && (pu += pn) < end) {
            const uint32_t bs = pu / per_slice, pr = pu - bs * per_slice, k0 = bs % p.slices * p.slice;
            left = min(p.slice, I - k0);
            ppieces = (left + 127) / 128;
            pn = min(per_slice - pr, end - pu);
            const Runs runs(pn, ppieces);
            pq = runs.begin(warp);
            pend = runs.begin(warp + 1);
            const uint32_t t = pq / ppieces;
            pp = pq - t * ppieces;
            src = m.w2 + ((uint64_t)expert_of(l, m.experts, bs / p.slices) * H + (pr + t) * 16 + lrow) * I + k0 + lchunk * 16;
        }
    };
    auto load = [&]() {
        if (pq < pend) {
            const uint32_t at = pp * 128 + lchunk * 16;
            const uint32_t bytes = at < left ? 16u : 0u;
            const uint32_t dst = ring_base + pslot * kTile;
            const int8_t* s = src + pp * 128;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t r = i * 4 + lrow;
                cp_async16(dst + r * 128 + ((lchunk ^ (r & 7)) * 16), bytes ? s + (uint64_t)i * 4 * I : m.w2, bytes);
            }
            if (++pp == ppieces) {
                pp = 0;
                src += (uint64_t)16 * I;
            }
            if (++pq == pend) settle();
        }
        cp_async_commit();
        if (++pslot == STAGES) pslot = 0;
    };
    if (begin < end) {
        settle();
#pragma unroll 1
        for (int i = 0; i < STAGES - 1; ++i) load();
    }
    griddep_wait();
    griddep_launch_dependents();
    if (begin == end) return;

    uint32_t slot = 0;
    uint32_t bs = begin / per_slice, ru = begin % per_slice;
    RowCopy copy;
    Block cur = block_at<NT>(l, m.experts, bs / p.slices);
    uint32_t k0 = bs % p.slices * p.slice, depth = min(p.slice, I - k0);
    copy.fetch(tid, p.hq, I, k0, depth, l.order + cur.r0, cur.count);
    const uint32_t g = lane >> 2, tig = lane & 3;
    for (uint32_t u = begin; u < end;) {
        const uint32_t r0 = cur.r0, count = cur.count;
        copy.finish(rows, row_pitch, p.hq, I, k0, depth, l.order + r0, count);
        __syncthreads();
        const uint32_t live = (count + 7) / 8, pieces = (depth + 127) / 128, here = min(per_slice - ru, end - u);
        if (u + here < end) {  // the next slice's rows, behind this one's products
            cur = block_at<NT>(l, m.experts, (bs + 1) / p.slices);
            k0 = (bs + 1) % p.slices * p.slice;
            depth = min(p.slice, I - k0);
            copy.fetch(tid, p.hq, I, k0, depth, l.order + cur.r0, cur.count);
        }
        auto finish = [&](uint32_t t, const int (&acc)[NT][4]) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t tok = nt * 8 + 2 * tig + c;
                    if (tok >= count) continue;
                    int32_t* at = p.acc + (uint64_t)l.order[r0 + tok] * H + (ru + t) * 16 + g;
                    if (p.slices > 1) {  // integers: exact in any order
                        atomicAdd(at, acc[nt][c]);
                        atomicAdd(at + 8, acc[nt][2 + c]);
                    } else {
                        at[0] = acc[nt][c];
                        at[8] = acc[nt][2 + c];
                    }
                }
        };
        const Runs runs(here, pieces);
        uint32_t q = runs.begin(warp), t = q / pieces, p0 = q - t * pieces;
        const uint32_t qe = runs.begin(warp + 1);
        int acc[NT][4];
        while (q < qe) {
            const uint32_t n = min(pieces - p0, qe - q);
            tile_product<NT, STAGES>(p0, n, live, ring_base, smem_u32(rows), row_pitch, slot, acc, load);
            if (n == pieces)
                finish(t, acc);
            else
                add_sums<NT, S::pitch>(sums + runs.place_of(warp, t) * S::tile_sums, acc, live);
            q += n;
            p0 = 0;
            ++t;
        }
        __syncthreads();
        const uint32_t cut = runs.cut_tile(warp);  // the tiles between two runs, a warp each
        if (cut != ~0u) {
            take_sums<NT, S::pitch>(sums + (warp - 1) * S::tile_sums, acc);
            finish(cut, acc);
        }
        // (the rows are read; the sums are zero before the next adds: the barrier behind the next rows)
        u += here;
        ++bs;
        ru = 0;
    }
    cp_async_wait<0>();
}

// out[t][i] = sum over the slots of w * float(acc) * (rs2 * s2), two outputs a thread.
template <typename T>
__global__ void __launch_bounds__(kThreads) moe_sum_kernel(Params p)
{
    griddep_launch_dependents();
    const MoeLayer& m = p.m;
    const uint32_t i = (blockIdx.x * kThreads + threadIdx.x) * 2, t = blockIdx.y;
    const bool on = i < m.hidden;
    constexpr uint32_t AHEAD = 8;
    // All but the sums is there before the product in front of this kernel is done: the layer's inputs, and the routes'
    // maxima, which that product waited for itself.
    float w[AHEAD];
    float2 sc[AHEAD];
    auto scales = [&](uint32_t k0) {
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k) {
            w[k] = 0.f;
            sc[k] = make_float2(0.f, 0.f);
            if (!on || k0 + k >= m.topk) continue;
            const uint32_t r = t * m.topk + k0 + k, e = (uint32_t)__ldg(m.topk_ids + r);
            if (e >= m.experts) continue;
            w[k] = __ldg(m.topk_w + r);
            const float rs = scale_of(__ldcg(p.top + r), m.qmax);
            const float* s = m.s2 + (uint64_t)e * m.hidden + i;
            sc[k] = make_float2(__fmul_rn(rs, __ldg(s)), __fmul_rn(rs, __ldg(s + 1)));
        }
    };
    scales(0);
    griddep_wait();
    if (!on) return;
    float2 sum = make_float2(0.f, 0.f);
    for (uint32_t k0 = 0; k0 < m.topk; k0 += AHEAD) {
        if (k0 > 0) scales(k0);
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k) {
            if (k0 + k >= m.topk) break;
            const uint32_t r = t * m.topk + k0 + k;
            if ((uint32_t)__ldg(m.topk_ids + r) >= m.experts) continue;
            const int2 a = __ldcg(reinterpret_cast<const int2*>(p.acc + (uint64_t)r * m.hidden + i));
            sum.x = fmaf(w[k], __fmul_rn((float)a.x, sc[k].x), sum.x);
            sum.y = fmaf(w[k], __fmul_rn((float)a.y, sc[k].y), sum.y);
        }
    }
    T* out = static_cast<T*>(m.out) + (uint64_t)t * m.hidden + i;
    out[0] = (T)sum.x;
    out[1] = (T)sum.y;
}

struct Ws {
    size_t xq, hq, rs1, top, h, acc, bytes;
};
Ws layout(uint32_t tokens, uint32_t hidden, uint32_t inter, uint32_t topk)
{
    const size_t r = (size_t)tokens * topk;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += (n + 255) / 256 * 256;
        return here;
    };
    Ws w;
    w.xq = take(r * hidden);
    w.hq = take(r * inter);
    w.rs1 = take(r * 4);
    w.top = take(r * 4);
    w.h = take(r * inter * 4);
    w.acc = take(r * hidden * 4);
    w.bytes = at;
    return w;
}

template <typename T, int NT, int STAGES>
cudaError_t run(Params& p, uint32_t num_sms, cudaStream_t st)
{
    using S = Smem<NT, STAGES>;
    const uint32_t routes = p.m.tokens * p.m.topk;
    static std::atomic<uint64_t> done1{0}, done2{0};
    cudaError_t e = allow_smem(moe_up_kernel<NT, STAGES>, kSmemMost, done1);
    if (e == cudaSuccess) e = allow_smem(moe_down_kernel<NT, STAGES>, kSmemMost, done2);
    if (e == cudaSuccess) e = launch_pdl(moe_quant_x_kernel<T>, dim3(routes), dim3(kThreads), 0, st, p);
    if (e == cudaSuccess)
        e = launch_pdl(moe_up_kernel<NT, STAGES>, dim3(num_sms), dim3(kThreads),
                       (size_t)S::total(p.m.hidden, p.m.experts, routes), st, p);
    if (e == cudaSuccess)
        e = launch_pdl(moe_quant_h_kernel, dim3((p.m.inter + 8 * kThreads - 1) / (8 * kThreads), routes), dim3(kThreads), 0, st,
                       p);
    if (e == cudaSuccess)
        e = launch_pdl(moe_down_kernel<NT, STAGES>, dim3(num_sms), dim3(kThreads),
                       (size_t)S::total(p.slice, p.m.experts, routes), st, p);
    if (e == cudaSuccess)
        e = launch_pdl(moe_sum_kernel<T>, dim3((p.m.hidden / 2 + kThreads - 1) / kThreads, p.m.tokens), dim3(kThreads), 0,
                       st, p);
    return e;
}

// The widest block of routes that the tokens call for and shared memory has room for, with as many stages as fit:
// a block too narrow for an expert's routes reads its weights again.  Narrow blocks gain from eleven stages (1 token:
// 64.1 us, with eight 65.7), wider ones do not.  Three stages under blocks of 32 lose more than reading twice (48 tokens,
// 32 experts, 8 slots, hidden 5120: 491 us against 433).
template <typename T, int NT>
cudaError_t pick(Params& p, uint32_t num_sms, cudaStream_t st)
{
    const uint32_t routes = p.m.tokens * p.m.topk, k = std::max(p.m.hidden, p.slice);
    if constexpr (NT == 1)
        if (Smem<NT, 11>::total(k, p.m.experts, routes) <= kSmemMost) return run<T, NT, 11>(p, num_sms, st);
    if (Smem<NT, 8>::total(k, p.m.experts, routes) <= kSmemMost) return run<T, NT, 8>(p, num_sms, st);
    if (Smem<NT, 5>::total(k, p.m.experts, routes) <= kSmemMost) return run<T, NT, 5>(p, num_sms, st);
    if constexpr (NT > 1) return pick<T, NT / 2>(p, num_sms, st);
    return cudaErrorInvalidValue;
}

// Routes of an expert at an even spread are about routes / experts; a block takes three standard deviations more (and no
// expert has more than the tokens, unless a token names it twice).  Narrow blocks leave room for a deeper ring: 24 tokens
// over 32 experts ran 107 us with blocks of 32 and five stages, 97 us with blocks of 16 and eight.
template <typename T>
cudaError_t run_type(Params& p, uint32_t num_sms, cudaStream_t st)
{
    const double mean = (double)p.m.tokens * p.m.topk / p.m.experts;
    const double most = std::min((double)p.m.tokens, mean + 3.0 * std::sqrt(mean) + 1.0);
    if (most <= 8) return pick<T, 1>(p, num_sms, st);
    if (most <= 16) return pick<T, 2>(p, num_sms, st);
    return pick<T, 4>(p, num_sms, st);
}

}  // namespace

size_t moe_layer_workspace(uint32_t tokens, uint32_t hidden, uint32_t inter, uint32_t topk)
{
    return layout(tokens, hidden, inter, topk).bytes;
}

cudaError_t launch_moe_layer(const MoeLayer& m, void* workspace, uint32_t num_sms, cudaStream_t st)
{
    const Ws w = layout(m.tokens, m.hidden, m.inter, m.topk);
    uint8_t* base = static_cast<uint8_t*>(workspace);
    Params p{};
    p.m = m;
    p.xq = reinterpret_cast<int8_t*>(base + w.xq);
    p.hq = reinterpret_cast<int8_t*>(base + w.hq);
    p.rs1 = reinterpret_cast<float*>(base + w.rs1);
    p.top = reinterpret_cast<uint32_t*>(base + w.top);
    p.h = reinterpret_cast<float*>(base + w.h);
    p.acc = reinterpret_cast<int32_t*>(base + w.acc);
    p.slices = (m.inter + kSliceMost - 1) / kSliceMost;
    p.slice = ((m.inter + p.slices - 1) / p.slices + 127) / 128 * 128;
    p.slices = (m.inter + p.slice - 1) / p.slice;
    return m.bf16 ? run_type<__nv_bfloat16>(p, num_sms, st) : run_type<__half>(p, num_sms, st);
}

}  // namespace b2sq
