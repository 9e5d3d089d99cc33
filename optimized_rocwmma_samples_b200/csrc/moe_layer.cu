// moe_layer.cu — a whole mixture-of-experts layer for a few tokens.
//
// For every route r = (token t, slot k) with expert e = topk_ids[t][k]:
//   xq, rs1 = smoothquant(x[t], smooth1[e])
//   [g | u] = float(w13[e] xq) * (rs1 * s13[e])
//   h       = g / (1 + exp(-g)) * u * smooth2[e];  hq, rs2 = its quantisation
//   d       = float(w2[e] hq) * (rs2 * s2[e])
//   out[t]  = sum over k of topk_w[t][k] * d, in slot order
// A route whose id is outside [0, experts) adds nothing.
//
// What bounds it is reading the weights of the experts that were chosen, once.
// Blocks of an expert's routes (up to 8 NT of them) meet its weight rows in
// units of 16 rows; every block of the grid (one an SM) takes an equal run of
// the units, which lie one after another in memory.  Weights stream through a
// ring of cp.async stages in which each of the eight warps keeps its own
// 16 x 128 byte tiles (every eighth of the unit's), so that no barrier stands
// between loading and multiplying; the routes' int8 rows lie in shared memory.
// mma.m16n8k32: weight rows are the 16, routes the 8 columns.  The warps' int32
// sums meet in shared memory by integer adds, one barrier a unit.
//
//   moe_up_kernel    quantises x for its expert, multiplies gate and up rows
//                    (8 + 8 a unit, so one thread has both), applies SwiGLU,
//                    leaves h in fp32 and the largest |h| it saw of each route
//   moe_down_kernel  starts streaming w2 before the first kernel is done, takes
//                    the maxima, quantises its slice of h, multiplies; slices of
//                    the inner dimension are added as integers (exact, any order)
//   moe_sum_kernel   scales, weighs and adds the slots
#include "common.cuh"
#include "kernels.h"
#include "sq_math.cuh"

#include <algorithm>
#include <atomic>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2sq {

namespace {

constexpr uint32_t kWarps = 8;
constexpr uint32_t kThreads = kWarps * 32;
constexpr uint32_t kTile = 2048;         // bytes of a warp's stage: 16 rows of 128
constexpr uint32_t kTilesMost = 2;
constexpr uint32_t kSliceMost = 4096;    // inner elements of h that a block of the second kernel holds at a time
constexpr uint32_t kSmemMost = 231424;   // dynamic shared memory: 227 KB, less 1 KB for what is static

struct Lists {
    uint16_t *first, *block, *order;  // [E + 1] first route and first block of an expert, [R] routes by expert
};

struct Params {
    MoeLayer m;
    float* h;        // [R][inter]
    float* part_max; // [blocks of the first kernel][R]
    float* rs2;      // [R]
    int32_t* acc;    // [R][hidden]
    uint32_t grid1, slices, slice;  // of the second kernel: slices of `slice` inner elements
    uint32_t tiles1, tiles2;        // row tiles of a unit: 2 where the pieces of one do not divide evenly among the warps
};

// Shared memory of both products: the ring, the routes' rows, the sums, the lists.
template <int NT, int STAGES>
struct Smem {
    static constexpr uint32_t ring = kWarps * STAGES * kTile;
    static constexpr uint32_t pitch = NT == 1 ? 8 : NT == 2 ? 24 : 40;  // ints of a row of sums: two-way bank conflicts at most
    static constexpr uint32_t sums = 2 * kTilesMost * 16 * pitch * 4;  // two units
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

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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

// Loads that stay where they are written, ahead of the asynchronous copies behind them.
__device__ __forceinline__ uint4 load16(const void* p)
{
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ float4 load16f(const float* p)
{
    float4 v;
    asm volatile("ld.global.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
    return v;
}

// Eight activations times their smooth scales, in fp32 (smoothquant's first step).
template <typename T>
__device__ __forceinline__ void smoothed(const uint4& w, const float4& s0, const float4& s1, float (&f)[8])
{
    const float2 a = pair_to_f2<T>(w.x), b = pair_to_f2<T>(w.y), c = pair_to_f2<T>(w.z), d = pair_to_f2<T>(w.w);
    f[0] = __fmul_rn(a.x, s0.x), f[1] = __fmul_rn(a.y, s0.y), f[2] = __fmul_rn(b.x, s0.z), f[3] = __fmul_rn(b.y, s0.w);
    f[4] = __fmul_rn(c.x, s1.x), f[5] = __fmul_rn(c.y, s1.y), f[6] = __fmul_rn(d.x, s1.z), f[7] = __fmul_rn(d.y, s1.w);
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
    __syncthreads();
    if (warp == 0)
        for (uint32_t base = 0; base < routes; base += 32) {
            const uint32_t r = base + lane;
            const uint32_t e = r < routes ? (uint32_t)__ldg(m.topk_ids + r) : 0xffffffffu;
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

// Equal runs of `total` units for `blocks` blocks: the first `rest` get one more.
struct Split {
    uint32_t each, rest;
    __device__ __forceinline__ Split(uint32_t total, uint32_t blocks) : each(total / blocks), rest(total % blocks) {}
    __device__ __forceinline__ uint32_t begin(uint32_t i) const { return i * each + min(i, rest); }
    __device__ __forceinline__ uint32_t block_of(uint32_t u) const
    {
        const uint32_t big = rest * (each + 1);
        return u < big ? u / (each + 1) : rest + (u - big) / each;
    }
};

// First of the 128-byte pieces of row tile `tile` that a warp takes: the unit's pieces, tile after tile, go round the warps.
__device__ __forceinline__ uint32_t first_piece(uint32_t warp, uint32_t tile, uint32_t pieces)
{
    return (warp - tile * pieces) & (kWarps - 1);
}

// A warp's share of a row tile: int32 products of its 16 weight rows with the block's routes over its pieces.
template <int NT, int STAGES, typename Next>
__device__ __forceinline__ void tile_product(uint32_t tile, uint32_t pieces, uint32_t live, uint32_t ring_base,
                                             uint32_t rows_base, uint32_t row_pitch, uint32_t& slot, int (&acc)[NT][4],
                                             Next&& next)
{
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const uint32_t arow = (lane & 7) + ((lane >> 3) & 1) * 8, asel = lane >> 4;
    const uint32_t brow = rows_base + (lane & 7) * row_pitch + (lane >> 3) * 16;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][i] = 0;
    for (uint32_t p = first_piece(warp, tile, pieces); p < pieces; p += kWarps) {
        cp_async_wait<STAGES - 2>();
        __syncwarp();
        // the slot that the last step freed takes the tile STAGES - 1 steps ahead
        next();
        const uint32_t a_at = ring_base + slot * kTile + arow * 128;
        if (++slot == STAGES) slot = 0;
        uint32_t a[4][4];
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q) ldsm4(a_at + (((q * 2 + asel) ^ (arow & 7)) * 16), a[q]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            if (nt == 0 || nt < live) {
                const uint32_t b_at = brow + nt * 8 * row_pitch + p * 128;
                uint32_t b[2][4];
                ldsm4(b_at, b[0]);
                ldsm4(b_at + 64, b[1]);
                mma_s8(acc[nt], a[0], b[0][0], b[0][1]);
                mma_s8(acc[nt], a[1], b[0][2], b[0][3]);
                mma_s8(acc[nt], a[2], b[1][0], b[1][1]);
                mma_s8(acc[nt], a[3], b[1][2], b[1][3]);
            }
    }
}

// Adds the warps' products into the unit's sums in shared memory (zero before).
template <int NT, uint32_t PITCH>
__device__ __forceinline__ void add_sums(int* sums, const int (&acc)[NT][4], uint32_t live)
{
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, tig = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
        if (nt == 0 || nt < live) {
            int* at = sums + g * PITCH + nt * 8 + 2 * tig;
            atomicAdd(at, acc[nt][0]);
            atomicAdd(at + 1, acc[nt][1]);
            atomicAdd(at + 8 * PITCH, acc[nt][2]);
            atomicAdd(at + 8 * PITCH + 1, acc[nt][3]);
        }
}

// Gate and up rows.  Units: block of routes x 8 inner elements.
template <typename T, int NT, int STAGES>
__global__ void __launch_bounds__(kThreads, 1) moe_up_kernel(Params p)
{
    using S = Smem<NT, STAGES>;
    extern __shared__ __align__(128) uint8_t moe_smem[];
    __shared__ float rs1[8 * NT];
    __shared__ uint32_t top[8 * NT];
    __shared__ float warp_max[kWarps];
    const MoeLayer& m = p.m;
    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const uint32_t routes = m.tokens * m.topk, H = m.hidden, I = m.inter;
    const uint32_t row_pitch = S::row_pitch(H);
    uint8_t* rows = moe_smem + S::ring;
    int* sums = reinterpret_cast<int*>(rows + S::rows(H));
    uint16_t* list = reinterpret_cast<uint16_t*>(reinterpret_cast<uint8_t*>(sums) + S::sums);
    const Lists l{list, list + m.experts + 1, list + 2 * (m.experts + 1)};

    griddep_wait();
    griddep_launch_dependents();
    make_lists(m, 8 * NT, l, reinterpret_cast<uint32_t*>(moe_smem));
    if (p.slices > 1)  // the second kernel's sums start from zero
        for (uint64_t i = (uint64_t)blockIdx.x * kThreads + tid; i < (uint64_t)routes * H / 4; i += (uint64_t)gridDim.x * kThreads)
            reinterpret_cast<int4*>(p.acc)[i] = make_int4(0, 0, 0, 0);
    for (uint32_t i = tid; i < S::sums / 4; i += kThreads) sums[i] = 0;

    const uint32_t tiles = p.tiles1;
    const uint32_t per_block = (I / 8 + tiles - 1) / tiles, total = l.block[m.experts] * per_block;
    const Split split(total, gridDim.x);
    const uint32_t begin = split.begin(blockIdx.x), end = split.begin(blockIdx.x + 1);
    if (begin == end) return;

    // producer: this warp's next piece (unit, row tile, piece) and its addresses
    const uint32_t pieces = (H + 127) / 128;
    const uint32_t ring_base = smem_u32(moe_smem) + warp * STAGES * kTile;
    const uint32_t lrow = lane / 8, lchunk = lane & 7;
    uint32_t pu = begin, pj = begin % per_block * tiles, pt = 0, pp = warp, pslot = 0;  // pj: row tile in the block
    const int8_t* src = nullptr;
    auto place = [&]() {
        const uint32_t e = expert_of(l, m.experts, pu / per_block);
        src = m.w13 + ((uint64_t)e * 2 * I + pj * 8 + lrow) * H + lchunk * 16;
    };
    // to the next piece of this warp, over row tiles and units in which it has none
    auto settle = [&]() {
        while (pu < end && (pp >= pieces || pj * 8 >= I)) {
            ++pj;
            if (++pt == tiles) {
                pt = 0;
                ++pu;
                if (pj * 8 >= I) pj = 0;
            }
            pp = first_piece(warp, pt, pieces);
            if (pu < end) {
                if (pj == 0)
                    place();
                else
                    src += (uint64_t)8 * H;
            }
        }
    };
    auto load = [&]() {
        if (pu < end) {
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
            pp += kWarps;
            settle();
        }
        cp_async_commit();
        if (++pslot == STAGES) pslot = 0;
    };
    place();
    settle();

    bool primed = false;
    uint32_t slot = 0, buf = 0;
    uint32_t b = begin / per_block, j = begin % per_block;
    for (uint32_t u = begin; u < end; ++b, j = 0) {
        const uint32_t e = expert_of(l, m.experts, b);
        const uint32_t r0 = l.first[e] + (b - l.block[e]) * 8 * NT;
        const uint32_t count = min(8u * NT, (uint32_t)l.first[e + 1] - r0);
        // Quantise the block's tokens, wpt warps each, so that a lane holds at most 64 values: they are read once, all
        // loads in flight together (behind the streaming weights a load takes microseconds), and for the first block
        // ahead of the weights.
        {
            uint32_t wpt = count > 4 ? 1 : count > 2 ? 2 : count > 1 ? 4 : 8;
            while (wpt * 2048 < H) wpt *= 2;
            const uint32_t per = kWarps / wpt;
            const float* sm = m.smooth1 + (uint64_t)e * H;
            const uint32_t start = (warp & (wpt - 1)) * 256 + lane * 8, stride = wpt * 256;
            for (uint32_t t0 = 0; t0 < count; t0 += per) {
                const uint32_t t = t0 + warp / wpt;
                const bool on = t < count;
                const T* x = static_cast<const T*>(m.x) + (uint64_t)(on ? l.order[r0 + t] / m.topk : 0) * m.x_stride;
                uint4 xw[8];
                float4 sw[8][2];
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    const uint32_t k = start + i * stride;
                    xw[i] = make_uint4(0, 0, 0, 0);
                    sw[i][0] = sw[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (on && k < H) {
                        xw[i] = load16(x + k);
                        sw[i][0] = load16f(sm + k);
                        sw[i][1] = load16f(sm + k + 4);
                    }
                }
                if (!primed) {
                    primed = true;
#pragma unroll 1
                    for (int i = 0; i < STAGES - 1; ++i) load();
                }
                float f[8][8], mx = 0.f;
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    smoothed<T>(xw[i], sw[i][0], sw[i][1], f[i]);
#pragma unroll
                    for (int c = 0; c < 8; ++c) mx = fmaxf(mx, fabsf(f[i][c]));
                }
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                __syncthreads();  // (also: the last block's rows, maxima and warp_max are read)
                if (lane == 0) warp_max[warp] = mx;
                __syncthreads();
                for (uint32_t w = warp & ~(wpt - 1); w < (warp & ~(wpt - 1)) + wpt; ++w) mx = fmaxf(mx, warp_max[w]);
                const float rs = row_scale_of(mx, m.qmax), inv = inv_scale_of(rs);
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    const uint32_t k = start + i * stride;
                    if (on && k < H) {
                        int8_t q[8];
#pragma unroll
                        for (int c = 0; c < 8; ++c) q[c] = quant1(f[i][c], inv, m.qmax);
                        *reinterpret_cast<uint2*>(rows + t * row_pitch + k) =
                            make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
                    }
                }
                if (on && lane == 0 && (warp & (wpt - 1)) == 0) {
                    rs1[t] = rs;
                    top[t] = 0;
                }
            }
            __syncthreads();
        }
        const uint32_t live = (count + 7) / 8;
        const uint32_t tok = tid / 8, jj = tid & 7;  // of the epilogue
        const bool mine = tok < count;
        const uint32_t route = mine ? l.order[r0 + tok] : 0;
        for (; j < per_block && u < end; ++j, ++u) {
            const uint32_t here = min(tiles, I / 8 - j * tiles);  // row tiles of this unit
            float sg[kTilesMost] = {}, su[kTilesMost] = {}, s2[kTilesMost] = {};
#pragma unroll
            for (uint32_t t = 0; t < kTilesMost; ++t)
                if (mine && t < here) {
                    const uint64_t at = (uint64_t)e * 2 * I + (j * tiles + t) * 8 + jj;
                    sg[t] = __ldg(m.s13 + at);
                    su[t] = __ldg(m.s13 + at + I);
                    s2[t] = __ldg(m.smooth2 + (uint64_t)e * I + (j * tiles + t) * 8 + jj);
                }
            int* sum = sums + buf * kTilesMost * 16 * S::pitch;
            buf ^= 1;
            for (uint32_t t = 0; t < here; ++t) {
                int acc[NT][4];
                tile_product<NT, STAGES>(t, pieces, live, ring_base, smem_u32(rows), row_pitch, slot, acc, load);
                add_sums<NT, S::pitch>(sum + t * 16 * S::pitch, acc, live);
            }
            __syncthreads();
            // (the other buffer's readers are past this barrier too: it is free and zero again)
#pragma unroll
            for (uint32_t t = 0; t < kTilesMost; ++t) {
                if (t >= here) break;
                int* at = sum + (t * 16 + jj) * S::pitch + tok;
                float hv = 0.f;
                if (mine) {
                    const float g = __fmul_rn((float)at[0], __fmul_rn(rs1[tok], sg[t]));
                    const float v = __fmul_rn((float)at[8 * S::pitch], __fmul_rn(rs1[tok], su[t]));
                    hv = g / (1.f + expf(-g)) * v * s2[t];
                    p.h[(uint64_t)route * I + (j * tiles + t) * 8 + jj] = hv;
                }
                if (tid < 64 * live) {  // cleared by the thread that read it
                    at[0] = 0;
                    at[8 * S::pitch] = 0;
                }
                float mx = fmaxf(fabsf(hv), 0.f);  // a NaN drops out, as in smoothquant
#pragma unroll
                for (int off = 4; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                if (mine && jj == 0) top[tok] = max(top[tok], __float_as_uint(mx));  // one thread a route
            }
        }
        // (every thread reads back what it wrote itself)
        if (mine && jj == 0) p.part_max[(uint64_t)blockIdx.x * routes + route] = __uint_as_float(top[tok]);
    }
    cp_async_wait<0>();
}

// Down rows.  Units: (block of routes, slice of the inner dimension) x 16 rows.
template <int NT, int STAGES>
__global__ void __launch_bounds__(kThreads, 1) moe_down_kernel(Params p)
{
    using S = Smem<NT, STAGES>;
    extern __shared__ __align__(128) uint8_t moe_smem[];
    __shared__ float inv2[8 * NT];
    const MoeLayer& m = p.m;
    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const uint32_t routes = m.tokens * m.topk, H = m.hidden, I = m.inter;
    const uint32_t row_pitch = S::row_pitch(p.slice);
    uint8_t* rows = moe_smem + S::ring;
    int* sums = reinterpret_cast<int*>(rows + S::rows(p.slice));
    uint16_t* list = reinterpret_cast<uint16_t*>(reinterpret_cast<uint8_t*>(sums) + S::sums);
    const Lists l{list, list + m.experts + 1, list + 2 * (m.experts + 1)};

    // before the wait: only what the layer's inputs say (the first kernel has waited for them)
    make_lists(m, 8 * NT, l, reinterpret_cast<uint32_t*>(moe_smem));
    for (uint32_t i = tid; i < S::sums / 4; i += kThreads) sums[i] = 0;
    const uint32_t tiles = p.tiles2;
    const uint32_t per_slice = (H / 16 + tiles - 1) / tiles, per_block = per_slice * p.slices;
    const uint32_t total = l.block[m.experts] * per_block;
    const Split split(total, gridDim.x);
    const uint32_t begin = split.begin(blockIdx.x), end = split.begin(blockIdx.x + 1);

    const uint32_t ring_base = smem_u32(moe_smem) + warp * STAGES * kTile;
    const uint32_t lrow = lane / 8, lchunk = lane & 7;
    uint32_t pu = begin, pr = begin % per_slice * tiles, pt = 0, pp = warp, pslot = 0;  // pr: row tile of the matrix
    const int8_t* src = nullptr;
    uint32_t left = 0, ppieces = 0;  // inner elements and pieces of the producer's slice
    auto place = [&]() {
        const uint32_t bs = pu / per_slice, e = expert_of(l, m.experts, bs / p.slices), k0 = bs % p.slices * p.slice;
        left = min(p.slice, I - k0);
        ppieces = (left + 127) / 128;
        src = m.w2 + ((uint64_t)e * H + pr * 16 + lrow) * I + k0 + lchunk * 16;
    };
    auto settle = [&]() {
        while (pu < end && (pp >= ppieces || pr * 16 >= H)) {
            ++pr;
            bool fresh = false;
            if (++pt == tiles) {
                pt = 0;
                ++pu;
                if (pr * 16 >= H) {
                    pr = 0;
                    fresh = true;
                }
            }
            if (pu < end) {
                if (fresh)
                    place();
                else
                    src += (uint64_t)16 * I;
            }
            pp = first_piece(warp, pt, ppieces);
        }
    };
    auto load = [&]() {
        if (pu < end) {
            const uint32_t at = pp * 128 + lchunk * 16;
            const uint32_t bytes = at < left ? 16u : 0u;
            const uint32_t dst = ring_base + pslot * kTile;
            const int8_t* s = src + pp * 128;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t r = i * 4 + lrow;
                cp_async16(dst + r * 128 + ((lchunk ^ (r & 7)) * 16), bytes ? s + (uint64_t)i * 4 * I : m.w2, bytes);
            }
            pp += kWarps;
            settle();
        }
        cp_async_commit();
        if (++pslot == STAGES) pslot = 0;
    };
    if (begin < end) {
        place();
        settle();
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) load();
    }
    griddep_wait();
    griddep_launch_dependents();
    if (begin == end) return;

    const uint32_t up_units = (I / 8 + p.tiles1 - 1) / p.tiles1;
    const Split up(l.block[m.experts] * up_units, p.grid1);
    uint32_t slot = 0, buf = 0;
    uint32_t bs = begin / per_slice, ru = begin % per_slice;
    for (uint32_t u = begin; u < end; ++bs, ru = 0) {
        const uint32_t b = bs / p.slices, k0 = bs % p.slices * p.slice, depth = min(p.slice, I - k0);
        const uint32_t e = expert_of(l, m.experts, b);
        const uint32_t r0 = l.first[e] + (b - l.block[e]) * 8 * NT;
        const uint32_t count = min(8u * NT, (uint32_t)l.first[e + 1] - r0);
        // the first 16 quads of h of each thread are in flight while the routes' scales are found
        const uint32_t quads = depth / 4, all = count * quads;  // depth is a multiple of 16
        float4 hv[16];
        auto fetch = [&](uint32_t i0) {
#pragma unroll
            for (uint32_t n = 0; n < 16; ++n) {
                const uint32_t i = i0 + n * kThreads;
                hv[n] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < all) {
                    const uint32_t t = i / quads;
                    hv[n] = load16f(p.h + (uint64_t)l.order[r0 + t] * I + k0 + (i - t * quads) * 4);
                }
            }
        };
        fetch(tid);
        __syncthreads();  // the last slice's rows are read
        {  // the largest of the maxima of the blocks that made a route's h
            const uint32_t c0 = up.block_of(b * up_units), c1 = up.block_of(b * up_units + up_units - 1);
            for (uint32_t t = warp; t < count; t += kWarps) {
                const uint32_t r = l.order[r0 + t];
                float mx = 0.f;
                for (uint32_t c = c0 + lane; c <= c1; c += 32) mx = fmaxf(mx, p.part_max[(uint64_t)c * routes + r]);
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                const float rs = row_scale_of(mx, m.qmax);
                if (lane == 0) {
                    inv2[t] = inv_scale_of(rs);
                    p.rs2[r] = rs;  // every block that needs it finds the same
                }
            }
        }
        __syncthreads();
        for (uint32_t i0 = tid;;) {
#pragma unroll
            for (uint32_t n = 0; n < 16; ++n) {
                const uint32_t i = i0 + n * kThreads;
                if (i < all) {
                    const uint32_t t = i / quads;
                    const float inv = inv2[t];
                    *reinterpret_cast<uint32_t*>(rows + t * row_pitch + (i - t * quads) * 4) =
                        pack4(quant1(hv[n].x, inv, m.qmax), quant1(hv[n].y, inv, m.qmax), quant1(hv[n].z, inv, m.qmax),
                              quant1(hv[n].w, inv, m.qmax));
                }
            }
            i0 += 16 * kThreads;
            if (i0 - tid >= all) break;
            fetch(i0);
        }
        __syncthreads();
        const uint32_t live = (count + 7) / 8, pieces = (depth + 127) / 128;
        for (; ru < per_slice && u < end; ++ru, ++u) {
            const uint32_t here = min(tiles, H / 16 - ru * tiles);
            int* sum = sums + buf * kTilesMost * 16 * S::pitch;
            buf ^= 1;
            for (uint32_t t = 0; t < here; ++t) {
                int acc[NT][4];
                tile_product<NT, STAGES>(t, pieces, live, ring_base, smem_u32(rows), row_pitch, slot, acc, load);
                add_sums<NT, S::pitch>(sum + t * 16 * S::pitch, acc, live);
            }
            __syncthreads();
            const uint32_t cells = 16 * here;
            for (uint32_t i = tid; i < cells * 8 * live; i += kThreads) {
                const uint32_t t = i / cells, row = i - t * cells;
                const int v = sum[row * S::pitch + t];
                sum[row * S::pitch + t] = 0;
                if (t < count) {
                    int32_t* at = p.acc + (uint64_t)l.order[r0 + t] * H + ru * tiles * 16 + row;
                    if (p.slices > 1)
                        atomicAdd(at, v);  // integers: exact in any order
                    else
                        *at = v;
                }
            }
        }
    }
    cp_async_wait<0>();
}

// out[t][i] = sum over the slots of w * float(acc) * (rs2 * s2)
template <typename T>
__global__ void __launch_bounds__(kThreads) moe_sum_kernel(Params p)
{
    griddep_wait();
    griddep_launch_dependents();
    const MoeLayer& m = p.m;
    const uint32_t i = (blockIdx.x * kThreads + threadIdx.x) * 2, t = blockIdx.y;
    if (i >= m.hidden) return;
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll 4
    for (uint32_t k = 0; k < m.topk; ++k) {
        const uint32_t r = t * m.topk + k;
        const uint32_t e = (uint32_t)__ldg(m.topk_ids + r);
        if (e >= m.experts) continue;
        const float w = __ldg(m.topk_w + r), rs = p.rs2[r];
        const int2 a = *reinterpret_cast<const int2*>(p.acc + (uint64_t)r * m.hidden + i);
        const float* s = m.s2 + (uint64_t)e * m.hidden + i;
        sum.x = fmaf(w, __fmul_rn((float)a.x, __fmul_rn(rs, __ldg(s))), sum.x);
        sum.y = fmaf(w, __fmul_rn((float)a.y, __fmul_rn(rs, __ldg(s + 1))), sum.y);
    }
    T* out = static_cast<T*>(m.out) + (uint64_t)t * m.hidden + i;
    out[0] = (T)sum.x;
    out[1] = (T)sum.y;
}

struct Ws {
    size_t h, part_max, rs2, acc, bytes;
};
Ws layout(uint32_t tokens, uint32_t hidden, uint32_t inter, uint32_t topk, uint32_t num_sms)
{
    const size_t r = (size_t)tokens * topk;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += (n + 255) / 256 * 256;
        return here;
    };
    Ws w;
    w.h = take(r * inter * 4);
    w.part_max = take(r * num_sms * 4);
    w.rs2 = take(r * 4);
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
    cudaError_t e = allow_smem(moe_up_kernel<T, NT, STAGES>, kSmemMost, done1);
    if (e == cudaSuccess) e = allow_smem(moe_down_kernel<NT, STAGES>, kSmemMost, done2);
    if (e == cudaSuccess)
        e = launch_pdl(moe_up_kernel<T, NT, STAGES>, dim3(num_sms), dim3(kThreads),
                       (size_t)S::total(p.m.hidden, p.m.experts, routes), st, p);
    if (e == cudaSuccess)
        e = launch_pdl(moe_down_kernel<NT, STAGES>, dim3(num_sms), dim3(kThreads),
                       (size_t)S::total(p.slice, p.m.experts, routes), st, p);
    if (e == cudaSuccess)
        e = launch_pdl(moe_sum_kernel<T>, dim3((p.m.hidden / 2 + kThreads - 1) / kThreads, p.m.tokens), dim3(kThreads), 0,
                       st, p);
    return e;
}

// The widest block of routes that the tokens call for and shared memory has room for, with eight stages or five:
// a block too narrow for an expert's routes reads its weights again.
template <typename T, int NT>
cudaError_t pick(Params& p, uint32_t num_sms, cudaStream_t st)
{
    const uint32_t routes = p.m.tokens * p.m.topk, k = std::max(p.m.hidden, p.slice);
    if (Smem<NT, 8>::total(k, p.m.experts, routes) <= kSmemMost) return run<T, NT, 8>(p, num_sms, st);
    if (Smem<NT, 5>::total(k, p.m.experts, routes) <= kSmemMost) return run<T, NT, 5>(p, num_sms, st);
    if constexpr (NT > 1) return pick<T, NT / 2>(p, num_sms, st);
    return cudaErrorInvalidValue;
}

template <typename T>
cudaError_t run_type(Params& p, uint32_t num_sms, cudaStream_t st)
{
    if (p.m.tokens <= 8) return pick<T, 1>(p, num_sms, st);
    if (p.m.tokens <= 16) return pick<T, 2>(p, num_sms, st);
    return pick<T, 4>(p, num_sms, st);
}

}  // namespace

size_t moe_layer_workspace(uint32_t tokens, uint32_t hidden, uint32_t inter, uint32_t, uint32_t topk, uint32_t num_sms)
{
    return layout(tokens, hidden, inter, topk, num_sms).bytes;
}

cudaError_t launch_moe_layer(const MoeLayer& m, void* workspace, uint32_t num_sms, cudaStream_t st)
{
    const Ws w = layout(m.tokens, m.hidden, m.inter, m.topk, num_sms);
    uint8_t* base = static_cast<uint8_t*>(workspace);
    Params p{};
    p.m = m;
    p.h = reinterpret_cast<float*>(base + w.h);
    p.part_max = reinterpret_cast<float*>(base + w.part_max);
    p.rs2 = reinterpret_cast<float*>(base + w.rs2);
    p.acc = reinterpret_cast<int32_t*>(base + w.acc);
    p.grid1 = num_sms;
    p.slices = (m.inter + kSliceMost - 1) / kSliceMost;
    p.slice = ((m.inter + p.slices - 1) / p.slices + 127) / 128 * 128;
    p.slices = (m.inter + p.slice - 1) / p.slice;
    p.tiles1 = (m.hidden + 127) / 128 % kWarps == 0 ? 1 : 2;
    p.tiles2 = p.slice / 128 % kWarps == 0 ? 1 : 2;
    return m.bf16 ? run_type<__nv_bfloat16>(p, num_sms, st) : run_type<__half>(p, num_sms, st);
}

}  // namespace b2sq
