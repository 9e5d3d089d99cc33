// kv4_attention.cu — attention of a few query tokens over the 4-bit cache.
//
// The queries of sequence b are its last tokens: query i of n sees positions
// below len - n + i + 1.  With keys K and values V as the cache stands for them:
//   s = scale * q . K,  p = exp(s - max s) / sum,  o = sum p V
// and, where asked, weight[head][position] += sum of p over the head's query
// heads and the queries.  A row that sees nothing gives 0.
//
// What bounds it is reading the cache (D/2 + D/16 bytes for a token's keys, as
// many for its values), so all query rows of a key head (its query heads times
// the queries) share one pass, 8 NT rows at a time, and nibbles become matrix
// operands with as few instructions as possible:
//  * A nibble masked out of a 16-bit word, q or 16 q, is the fp16 subnormal
//    q 2^-24 or q 2^-20.  mma.m16n8k16 takes subnormals as they are, so one AND
//    turns two nibbles into two operands (and a shift by 8 serves the word's
//    upper half).  The powers of two, the group's step and its base are applied
//    to the sums: q.K over a group = s * sum(q4 q) + z * sum(q).
//  * Scores: K is the 16 x 16 operand (16 tokens, 16 channels of one word
//    position), the query rows are the 8 columns, prepared once in that order
//    as fp16 scaled by a power of two that brings the row's largest to [2^9, 2^10)
//    (exact, but for channels below 2^-20 (fp16) or 2^-23 (bf16) of the largest,
//    which are off by up to 2^-30 of it).
//  * Output: V^T is the 16 x 16 operand; ldmatrix.trans moves whole 16-bit
//    words (4 channels of a token), which is the transposition needed.  The
//    probabilities, times the token's step over a running power of two of the
//    group, are rounded to fp16 (11 bits; the result has 8 or 11) and turned
//    into the other operand by movmatrix.  sum(p z) is kept apart in fp32.
//  * The matrix unit cuts its fp32 sums off instead of rounding them, and nibbles
//    are never negative: left alone the sums shrink by about 2^-23 a product,
//    and sum(p z), of the other sign, leaves that a large part of the result.
//    So every 32 products an amount known exactly, close to 8 steps times the
//    sum of p, moves from the sums to sum(p z): they stay about their centre,
//    where what is cut off cancels (64 x 131072 tokens, fp16: off by 2.2e-4 of
//    the result, 2.1e-3 without; rounding the result is 2.2e-4.  It takes 2 to
//    5% of the time; 8 steps taken off by a product of their own took 14%).
//
// Work is split evenly over the grid in chunks of 16 tokens, whatever the
// lengths: the (sequence, head, row block) items lie one after another on a
// line of chunks and every block takes an equal piece of it.  Blocks that get
// part of an item leave their maxima, sums and outputs in the workspace, and a
// second kernel joins them in a fixed order (and adds up the weights from the
// scores that the first one left there).  In a block each of the four warps
// streams its own chunks through a ring of cp.async stages, with no barrier
// until the item's end.
//
// 2 x 100001 tokens, 64 heads over 8 of 128 channels: 56 us (221 MB, 3.9 TB/s),
// with about 290 warp instructions for 16 tokens of a head, 80 of them masks,
// beside the bytes; neither is full (0.54 instructions a cycle): with three warps
// a scheduler the latencies of masks and products show.  16 x 4000, 32 heads: 24
// us, 15 of which do not depend on the lengths (start, joins, second kernel); 48
// x 8192 with weights 100 us, 25 of them the second kernel's reading of the
// scores; 1 x 257: 11.8 us.
#include "kv4.cuh"
#include "sq_math.cuh"

#include <algorithm>
#include <type_traits>

namespace b2sq {

namespace {

// Tokens of a block's share: fewer leave too little to do between its start and its join.  Shorter items have a block
// each while there are blocks (4 x 7 tokens, 4 key heads: one after another they took 27 us, side by side 9).
constexpr uint32_t kMinTokens = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kRun = 32;           // products between two centrings of the sums (16 gave the same error)
constexpr float kSample = 1.f / 256.f;  // keeps a sample's sum in fp16: 32 products, 8 lanes, p times step at most 2^15

struct AttnParams {
    Kv4Cache c;
    Kv4Seqs s;
    const void* q;
    void* out;
    uint64_t q_stride;
    uint32_t heads, group;
    uint32_t first_query, max_queries, all_queries;  // of a sequence's: the first and the number of this launch, the call's
    uint32_t row_pad;                                // group * max_queries rounded up to 4
    float scale;
    uint32_t chunk;  // tokens a warp takes at a time: 16 or 32
    uint32_t items;  // (sequence, head, row block) at most
    float2* stats;         // [batch * kv_heads][row_pad] (max, sum) of items that one block did whole
    float* part_o;         // [2 * blocks][8 NT][D]
    float2* part_ml;       // [2 * blocks][8 NT]
    float* scores;         // [batch * kv_heads][positions][row_pad], for the weights
};

// Warps of a block, and blocks a SM that registers and shared memory leave room for.
template <int D, int NT, int CH>
constexpr uint32_t attn_warps()
{
    return 4;  // one a scheduler: five were slower (60.5 us against 57.5 at 2 x 100001 tokens)
}
template <int D, int NT, int CH>
constexpr uint32_t attn_blocks()
{
    if (CH == 2) return D == 64 ? 4 : 3;
    return D == 64 ? (NT == 1 ? 5 : 4) : D == 128 ? (NT == 1 ? 4 : 3) : (NT == 1 ? 3 : 2);
}
constexpr uint32_t kMaxBlocks = 5;

template <int D, int NT, int CH>
struct AttnSmem {
    static constexpr uint32_t rows = 8 * NT;
    static constexpr uint32_t warps = attn_warps<D, NT, CH>();
    static constexpr uint32_t data = CH * 16 * D / 2;               // a chunk's key nibbles
    static constexpr uint32_t scales = CH * 16 * (D / 64) * 4;      // and their steps and bases
    static constexpr uint32_t stage = 2 * (data + scales);
    static constexpr uint32_t stages = D == 64 ? (CH == 2 ? 3 : 5) : 3;
    static constexpr uint32_t ring = warps * stages * stage;
    static constexpr uint32_t q = rows * D * 2;
    static constexpr uint32_t pitch = D + 2;  // of a row in the join of the warps
    static constexpr uint32_t merge = warps * 8 * pitch * 4;
    static constexpr bool early = D < 256;  // room for the join beside the ring, so that the next piece's loads need not wait
    static_assert(early || merge <= ring, "ring too small for the join");
    static constexpr uint32_t fixed = ring + q + (early ? merge : 0);
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x)
{
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
    return d;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <uint32_t N>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[N])
{
    if constexpr (N == 1) {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x, w[1] = v.y;
    } else {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
}
// Words j of four nibbles each become fp16 subnormals: nibbles 0 and 2 stand for q 2^-24, 1 and 3 for q 2^-20.
template <int J>
__device__ __forceinline__ uint32_t nibbles(uint32_t w)
{
    return (J < 2 ? w : w >> 8) & ((J & 1) ? 0x00f000f0u : 0x000f000fu);
}

struct SeqShape {
    uint32_t len, n, start, queries, vis, chunks, blocks;
};
// start, queries: the rows of this launch; vis: positions with a place in the table; an empty sequence has one chunk in which nothing is seen
__device__ __forceinline__ SeqShape seq_shape(const AttnParams& a, uint32_t b, uint32_t rows)
{
    SeqShape s;
    s.len = kv4_len(a.s, b);
    s.n = kv4_new_rows(a.s, b, s.start);
    s.start += a.first_query;
    const uint32_t upto = min(s.n, a.all_queries);
    s.queries = upto > a.first_query ? min(upto - a.first_query, a.max_queries) : 0;
    s.vis = min(s.len, kv4_cap(a.c, a.s));
    s.chunks = max(1u, (s.vis + a.chunk - 1) / a.chunk);
    s.blocks = (s.queries * a.group + rows - 1) / rows;
    return s;
}
// For the values, two operands a byte: nibble 0 (J even), and the byte itself, nibble 0 + 16 nibble 1 (J odd): the sums
// over nibble 1 come from the difference in the end, which saves a mask.  `hi`: the upper bytes of w's halves.
template <int J>
__device__ __forceinline__ uint32_t value_bits(uint32_t w, uint32_t hi)
{
    if constexpr (J == 0) return w & 0x000f000fu;
    if constexpr (J == 1) return w & 0x00ff00ffu;
    if constexpr (J == 2) return hi & 0x000f000fu;
    return hi;
}

// Equal pieces of `total` chunks for `blocks` blocks: the first `rest` get one more.
struct Split {
    uint32_t blocks, each, rest;
    __device__ __forceinline__ Split(uint32_t total, uint32_t grid, uint32_t chunk, uint32_t items)
    {
        blocks = max(1u, min(grid, max(total / (kMinTokens / chunk), min(total, items))));
        each = total / blocks;
        rest = total - each * blocks;
    }
    __device__ __forceinline__ uint32_t begin(uint32_t i) const { return i * each + min(i, rest); }
    __device__ __forceinline__ uint32_t block_of(uint32_t unit) const
    {
        const uint32_t big = rest * (each + 1);
        return unit < big ? unit / (each + 1) : rest + (unit - big) / each;
    }
};

// First chunk of every sequence on the line, into shared memory [batch + 1] (and, where asked, the chunks of its items
// [batch]); all threads of the block.
template <uint32_t THREADS>
__device__ __forceinline__ void lay_out(const AttnParams& a, uint32_t rows, uint32_t* ustart, uint32_t* part,
                                        uint32_t* chunks = nullptr)
{
    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    uint32_t carry = 0;
    for (uint32_t base = 0; base < a.s.batch; base += THREADS) {
        const uint32_t b = base + tid;
        uint32_t v = 0, here = 1;
        if (b < a.s.batch) {
            const SeqShape sh = seq_shape(a, b, rows);
            here = sh.chunks;
            v = sh.chunks * sh.blocks * a.c.kv_heads;
        }
        uint32_t incl = v;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= (uint32_t)off) incl += t;
        }
        if (lane == 31) part[warp] = incl;
        __syncthreads();
        uint32_t before = carry;
        for (uint32_t w = 0; w < THREADS / 32; ++w) {
            if (w < warp) before += part[w];
            carry += part[w];
        }
        if (b < a.s.batch) {
            ustart[b] = before + incl - v;
            if (chunks) chunks[b] = here;
        }
        __syncthreads();
    }
    if (tid == 0) ustart[a.s.batch] = carry;
    __syncthreads();
}
// The last sequence that starts at or before `unit` (empty ones share their start with the next).
__device__ __forceinline__ uint32_t seq_of(const uint32_t* ustart, uint32_t batch, uint32_t unit)
{
    uint32_t lo = 0, hi = batch;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (ustart[mid] <= unit)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

template <typename T, int D, int NT, int CH>
__global__ void __launch_bounds__(attn_warps<D, NT, CH>() * 32, attn_blocks<D, NT, CH>()) kv4_attention_kernel(AttnParams a)
{
    using S = AttnSmem<D, NT, CH>;
    constexpr uint32_t kWarps = S::warps, kThreads = kWarps * 32;
    constexpr uint32_t CHUNK = 16 * CH, NG = D / 64, CPR = D / 32, ROWS = 8 * NT, STAGES = S::stages, SC = S::scales / 16;
    // fp16 results want more bits of the probabilities than fp16 has: a second operand holds what the first leaves
    constexpr bool SPLIT = std::is_same<T, __half>::value;
    extern __shared__ __align__(16) uint8_t at_smem[];
    uint8_t* ring = at_smem;
    __half* q_frag = reinterpret_cast<__half*>(at_smem + S::ring);  // [NT][NG][2][32 lanes] x 16 bytes
    float* merge = reinterpret_cast<float*>(S::early ? at_smem + S::ring + S::q : ring);  // [kWarps][8][pitch]
    uint32_t* ustart = reinterpret_cast<uint32_t*>(at_smem + S::fixed);  // [batch + 1]
    __shared__ float row_mul[ROWS], row_sum[ROWS][NG];
    __shared__ int row_vis[ROWS];
    __shared__ float2 warp_ml[kWarps][ROWS];
    __shared__ uint32_t scan_part[kWarps];

    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31, g = lane >> 2, tig = lane & 3;
    griddep_wait();
    griddep_launch_dependents();

    lay_out<kThreads>(a, ROWS, ustart, scan_part);
    const uint32_t total = ustart[a.s.batch];
    const Split split(total, gridDim.x, CHUNK, a.items);
    if (blockIdx.x >= split.blocks || total == 0) return;
    const uint32_t begin = split.begin(blockIdx.x), end = split.begin(blockIdx.x + 1);

    const uint32_t page_chunks = a.c.page_size / CHUNK;
    const uint32_t ring_base = smem_u32(ring) + warp * STAGES * S::stage;
    // A piece of an item: what of it is this block's, and of that this warp's (an even share, one chunk after another).
    struct Piece {
        SeqShape sh;
        uint32_t b, head, block, c0, c1, wc0, wc1, all_rows;
    };
    uint32_t seq = seq_of(ustart, a.s.batch, begin);
    auto piece_at = [&](uint32_t unit) {
        while (ustart[seq + 1] <= unit) ++seq;
        Piece p;
        p.b = seq;
        p.sh = seq_shape(a, seq, ROWS);
        const uint32_t in_seq = unit - ustart[seq], item = in_seq / p.sh.chunks;
        p.c0 = in_seq - item * p.sh.chunks;
        p.head = item / p.sh.blocks;
        p.block = item - p.head * p.sh.blocks;
        p.c1 = min(p.sh.chunks, p.c0 + (end - unit));
        p.all_rows = p.sh.queries * a.group;
        p.wc0 = p.c0 + (p.c1 - p.c0) * warp / kWarps;
        p.wc1 = p.c0 + (p.c1 - p.c0) * (warp + 1) / kWarps;
        return p;
    };
    // this warp's query rows of a piece, on their way (ahead of the piece's keys: behind them a load takes long)
    constexpr uint32_t QROWS = ROWS / kWarps;
    T qv[QROWS][D / 32];
    auto fetch_rows = [&](const Piece& p) {
#pragma unroll
        for (uint32_t i = 0; i < QROWS; ++i) {
            const uint32_t row = p.block * ROWS + warp + i * kWarps;
            const uint32_t qi = row / a.group, qh = p.head * a.group + row % a.group;
            const T* src = static_cast<const T*>(a.q) + (uint64_t)(p.sh.start + qi) * a.q_stride + (uint64_t)qh * D;
#pragma unroll
            for (uint32_t j = 0; j < D / 32; ++j) qv[i][j] = row < p.all_rows ? src[lane + 32 * j] : T(0.f);
        }
    };
    // loads run ahead of the computation by STAGES - 1 chunks, and page ids by one page
    uint32_t lc = 0, lend = 0, lslot = 0, left = 0;  // next chunk, the last one, its ring slot, chunks left on its page
    uint32_t valid = 0;                              // bit i: the chunk loaded i loads ago has a page
    uint32_t page_at = 0, page_end = 0, lskip = 0;
    int32_t page = -1, next_page = -1;
    const int32_t* ltable = nullptr;
    const uint8_t *kp = nullptr, *vp = nullptr, *sp = nullptr;
    uint64_t head_row = 0;
    auto load = [&]() {
        valid <<= 1;
        if (lc < lend) {
            if (left == 0) {
                left = page_chunks - lskip;
                page = next_page;
                ++page_at;
                next_page = page_at < page_end ? __ldg(ltable + page_at) : -1;
                const uint64_t row = (uint64_t)(uint32_t)page * a.c.kv_heads * a.c.page_size + head_row + lskip * CHUNK;
                lskip = 0;
                kp = a.c.k + row * (D / 2) + lane * 16;
                vp = a.c.v + row * (D / 2) + lane * 16;
                sp = static_cast<const uint8_t*>(lane < SC ? a.c.k_scale : a.c.v_scale) + row * (NG * 4) +
                     (lane < SC ? lane : lane - SC) * 16;
            }
            if ((uint32_t)page < a.c.pages) {
                valid |= 1;
                const uint32_t dst = ring_base + lslot * S::stage;
#pragma unroll
                for (uint32_t i = 0; i < S::data / 512; ++i) {
                    const uint32_t u = i * 32 + lane, r = u / CPR, ch = u % CPR;
                    const uint32_t to = r * CPR + (ch ^ ((r / (8 / CPR)) & (CPR - 1)));
                    cp_async16(dst + to * 16, kp + i * 512);
                    cp_async16(dst + S::data + to * 16, vp + i * 512);
                }
                if (lane < 2 * SC) cp_async16(dst + 2 * S::data + lane * 16, sp);
            }
            kp += S::data;
            vp += S::data;
            sp += S::scales;
            --left;
            ++lc;
        }
        cp_async_commit();
        if (++lslot == STAGES) lslot = 0;
    };
    auto begin_loads = [&](const Piece& p) {
        lc = p.wc0;
        lend = p.wc1;
        left = 0;
        page_at = lc / page_chunks;
        lskip = lc - page_at * page_chunks;
        page_end = p.sh.vis == 0 ? 0 : (p.sh.vis - 1) / a.c.page_size + 1;
        ltable = a.s.page_table + (uint64_t)p.b * a.s.max_pages;
        head_row = (uint64_t)p.head * a.c.page_size;
        next_page = page_at < page_end ? __ldg(ltable + page_at) : -1;
#pragma unroll 1
        for (uint32_t i = 0; i < STAGES - 1; ++i) load();
    };

    Piece cur = piece_at(begin);
    fetch_rows(cur);
    uint32_t slot = lslot;
    begin_loads(cur);
    for (uint32_t unit = begin;;) {
        const SeqShape sh = cur.sh;
        const uint32_t b = cur.b, head = cur.head, block = cur.block, all_rows = cur.all_rows, wc0 = cur.wc0, wc1 = cur.wc1;
        const bool whole = cur.c0 == 0 && cur.c1 == sh.chunks;
        // the rows become operands (the last piece's are no longer read: the warps have met since)
#pragma unroll
        for (uint32_t i = 0; i < QROWS; ++i) {
            const uint32_t r = warp + i * kWarps, row = block * ROWS + r;
            float v[D / 32], mx = 0.f;
#pragma unroll
            for (uint32_t j = 0; j < D / 32; ++j) {
                v[j] = (float)qv[i][j];
                mx = fmaxf(mx, fabsf(v[j]));
            }
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            // 2^(9 - exponent of the largest), 2^127 at most; none for rows with an infinity
            const int ex = (int)(__float_as_uint(mx) >> 23);
            const int shift = ex == 255 ? 0 : min(136 - ex, 127);
            const float f = __uint_as_float((uint32_t)(127 + shift) << 23);
            const float back = __uint_as_float(shift == 127 ? 1u << 22 : (uint32_t)(127 - shift) << 23);  // 1 / f
            // What brings the row's products back, below 2^76: there a softmax is 0 or 1, since products that differ do so
            // by 2^-48 or more, and the scores stay finite.
            const float mul = fminf(fmaxf(a.scale * back * kLog2e, -7.55578637e22f), 7.55578637e22f);
#pragma unroll
            for (uint32_t c = 0; c < D / 32; ++c) {
                // channel 32 c + lane: word position j, k half, operand register and lane
                const uint32_t gr = c / 2, cb = c & 1, t4 = lane / 8, y = lane & 7, j = y & 3, hi = y >> 2;
                const uint32_t at = ((((r / 8) * NG + gr) * 2 + j / 2) * 32 + (r & 7) * 4 + t4) * 8 + (j & 1) * 4 + cb * 2 + hi;
                q_frag[at] = __float2half_rn(v[c] * ((j & 1) ? f * 0.0625f : f));
            }
#pragma unroll
            for (uint32_t gr = 0; gr < NG; ++gr) {
                float sum = v[2 * gr] * f + v[2 * gr + 1] * f;
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                if (lane == 0) row_sum[r][gr] = sum * mul;
            }
            if (lane == 0) {
                row_mul[r] = mul * 16777216.f;
                // rows that are not there see everything (their columns are not used), so that they mask nothing
                row_vis[r] = row < all_rows
                                 ? (int)max((int64_t)0, min((int64_t)sh.vis, (int64_t)sh.len - sh.n + a.first_query + row / a.group + 1))
                                 : (int)sh.vis;
            }
        }
        __syncthreads();
        float mul[NT][2], qsum[NT][2][NG];
        int vis[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t r = nt * 8 + 2 * tig + x;
                mul[nt][x] = row_mul[r];
                vis[nt][x] = row_vis[r];
#pragma unroll
                for (uint32_t gr = 0; gr < NG; ++gr) qsum[nt][x][gr] = row_sum[r][gr];
            }
        // positions that all rows see
        const int least = __reduce_min_sync(0xffffffffu, lane < ROWS ? row_vis[lane % ROWS] : 0x7fffffff);

        float o[NG][4][NT][4] = {};
        float m[NT][2], l[NT][2], zs[NT][2][NG];  // m: 0 until the row has seen a token
        float ref[NG];                            // 2^8 / the power of two that a group's steps are taken over
        __half2 part_p[NG][NT];                   // half of the tokens' p times step since the last centring
        uint32_t seen = 0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                m[nt][x] = 0.f;
                l[nt][x] = 0.f;
#pragma unroll
                for (uint32_t gr = 0; gr < NG; ++gr) zs[nt][x][gr] = 0.f;
            }
#pragma unroll
        for (uint32_t gr = 0; gr < NG; ++gr) {
            ref[gr] = 4294967296.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) part_p[gr][nt] = __half2(0.f, 0.f);
        }

        const uint32_t tok = (lane & 7) + ((lane >> 3) & 1) * 8;  // ldmatrix row of this lane
        const uint32_t sw = (tok / (8 / CPR)) & (CPR - 1);
        const uint32_t mat = ring_base + tok * CPR * 16;
        float* score_at = a.scores ? a.scores + (((uint64_t)b * a.c.kv_heads + head) * kv4_cap(a.c, a.s) + wc0 * CHUNK + g) * a.row_pad + block * ROWS + 2 * tig
                                   : nullptr;

        // one chunk of 16 tokens; FULL: every row sees all of them
        auto step = [&](uint32_t c, uint32_t slot, auto full_tag) {
            constexpr bool FULL = decltype(full_tag)::value;
            const uint32_t base = mat + slot * S::stage;
            const uint8_t* stage = ring + (warp * STAGES + slot) * S::stage;
            const int t0 = (int)(c * CHUNK + g);
            bool see[CH][NT][4];
            float s[CH][NT][4];  // score - m
            uint32_t vw[CH][2][NG];  // the values' steps and bases
            float top = -INFINITY;
            float acc[CH][NG][NT][4];
#pragma unroll
            for (uint32_t gr = 0; gr < NG; ++gr) {
                uint32_t w[CH][4];
#pragma unroll
                for (int ch = 0; ch < CH; ++ch) ldsm4(base + ch * 8 * D + ((gr * 2 + (lane >> 4)) ^ sw) * 16, w[ch]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint4* qf = reinterpret_cast<const uint4*>(q_frag) + ((nt * NG + gr) * 2) * 32 + lane;
                    const uint4 q0 = qf[0], q1 = qf[32];
#pragma unroll
                    for (int ch = 0; ch < CH; ++ch) {
                        const uint32_t(&k)[4] = w[ch];
                        float(&d)[4] = acc[ch][gr][nt];
                        mma_f16_first(d, nibbles<0>(k[0]), nibbles<0>(k[1]), nibbles<0>(k[2]), nibbles<0>(k[3]), q0.x, q0.y);
                        mma_f16(d, nibbles<1>(k[0]), nibbles<1>(k[1]), nibbles<1>(k[2]), nibbles<1>(k[3]), q0.z, q0.w);
                        mma_f16(d, nibbles<2>(k[0]), nibbles<2>(k[1]), nibbles<2>(k[2]), nibbles<2>(k[3]), q1.x, q1.y);
                        mma_f16(d, nibbles<3>(k[0]), nibbles<3>(k[1]), nibbles<3>(k[2]), nibbles<3>(k[3]), q1.z, q1.w);
                    }
                }
            }
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) {
                // thread: tokens g and g + 8, rows 2 tig and 2 tig + 1 of every eight
                float2 ksz[2][NG];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t kw[NG];
                    lds_words<NG>(stage + 2 * S::data + (ch * 16 + g + 8 * h) * NG * 4, kw);
                    lds_words<NG>(stage + 2 * S::data + S::scales + (ch * 16 + g + 8 * h) * NG * 4, vw[ch][h]);
#pragma unroll
                    for (uint32_t gr = 0; gr < NG; ++gr) h2_to_f2(kw[gr], ksz[h][gr].x, ksz[h][gr].y);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int h = i >> 1, x = i & 1;
                        float dot = acc[ch][0][nt][i] * ksz[h][0].x, off = fmaf(qsum[nt][x][0], ksz[h][0].y, -m[nt][x]);
#pragma unroll
                        for (uint32_t gr = 1; gr < NG; ++gr) {
                            dot = fmaf(acc[ch][gr][nt][i], ksz[h][gr].x, dot);
                            off = fmaf(qsum[nt][x][gr], ksz[h][gr].y, off);
                        }
                        see[ch][nt][i] = FULL || t0 + 16 * ch + 8 * h < vis[nt][x];
                        s[ch][nt][i] = see[ch][nt][i] ? fmaf(dot, mul[nt][x], off) : -INFINITY;
                        top = fmaxf(top, s[ch][nt][i]);
                    }
                if (score_at) {
                    float* sp_at = score_at + ch * 16 * a.row_pad;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        // (the last chunk may reach past the table by its second half)
                        if (block * ROWS + nt * 8 + 2 * tig < a.row_pad && (CH == 1 || c * CHUNK + ch * 16 < sh.vis)) {
                            *reinterpret_cast<float2*>(sp_at + nt * 8) =
                                make_float2(s[ch][nt][0] + m[nt][0], s[ch][nt][1] + m[nt][1]);
                            *reinterpret_cast<float2*>(sp_at + 8 * a.row_pad + nt * 8) =
                                make_float2(s[ch][nt][2] + m[nt][0], s[ch][nt][3] + m[nt][1]);
                        }
                }
            }
            // largest steps of the groups (unseen tokens may hold anything; a NaN drops out)
            bool wide = false;
#pragma unroll
            for (uint32_t gr = 0; gr < NG; ++gr) {
                __half2 hm = __habs2(*reinterpret_cast<const __half2*>(&vw[0][0][gr]));
#pragma unroll
                for (int i = 1; i < 2 * CH; ++i)
                    hm = __hmax2(hm, __habs2(*reinterpret_cast<const __half2*>(&vw[i / 2][i & 1][gr])));
                wide |= __low2float(hm) * ref[gr] > 512.f;
            }
            // p may reach 2^6 and a step twice its power of two before the references are moved
            if (__any_sync(0xffffffffu, top > 6.f || wide || seen != (1u << (2 * NT)) - 1)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float mx = -INFINITY;
#pragma unroll
                        for (int ch = 0; ch < CH; ++ch) mx = fmaxf(mx, fmaxf(s[ch][nt][x], s[ch][nt][2 + x]));
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                        const uint32_t bit = 1u << (nt * 2 + x);
                        if (mx > 0.f || (!(seen & bit) && mx > -INFINITY)) {
                            const float f = (seen & bit) ? ex2(-mx) : 0.f;
                            seen |= bit;
                            m[nt][x] += mx;
#pragma unroll
                            for (int ch = 0; ch < CH; ++ch) {
                                s[ch][nt][x] -= mx;
                                s[ch][nt][2 + x] -= mx;
                            }
                            l[nt][x] *= f;
#pragma unroll
                            for (uint32_t gr = 0; gr < NG; ++gr) {
                                zs[nt][x][gr] *= f;
                                part_p[gr][nt] = __half2(0.f, 0.f);
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    o[gr][j][nt][x] *= f;
                                    o[gr][j][nt][2 + x] *= f;
                                }
                            }
                        }
                    }
#pragma unroll
                for (uint32_t gr = 0; gr < NG; ++gr) {
                    float mx = 0.f;
#pragma unroll
                    for (int ch = 0; ch < CH; ++ch)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float st = fabsf(__low2float(*reinterpret_cast<const __half2*>(&vw[ch][h][gr])));
                            if (t0 + 16 * ch + 8 * h < (int)sh.vis && st < INFINITY) mx = fmaxf(mx, st);
                        }
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                    if (mx * ref[gr] > 512.f) {
                        const float fresh = __uint_as_float((262u - (__float_as_uint(mx) >> 23)) << 23);
                        const float f = fresh / ref[gr];
                        ref[gr] = fresh;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) part_p[gr][nt] = __half2(0.f, 0.f);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int i = 0; i < 4; ++i) o[gr][j][nt][i] *= f;
                    }
                }
            }
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) {
                // probabilities
                float pw[2][NG], vz[2][NG];  // steps over the group's power of two, and bases
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (uint32_t gr = 0; gr < NG; ++gr) {
                        float st;
                        h2_to_f2(vw[ch][h][gr], st, vz[h][gr]);
                        pw[h][gr] = st * ref[gr];
                    }
                uint32_t pb[NG][NT][2];
                [[maybe_unused]] uint32_t pb2[SPLIT ? NG : 1][NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float p[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        p[i] = ex2(s[ch][nt][i]);  // 0 where unseen
                        l[nt][i & 1] += p[i];
                    }
#pragma unroll
                    for (uint32_t gr = 0; gr < NG; ++gr) {
                        float pv[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int h = i >> 1, x = i & 1;
                            if (FULL || see[ch][nt][i]) zs[nt][x][gr] = fmaf(p[i], vz[h][gr], zs[nt][x][gr]);
                            pv[i] = FULL || see[ch][nt][i] ? p[i] * pw[h][gr] : 0.f;
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t w = f2_to_pair<__half>(pv[2 * h], pv[2 * h + 1]);
                            pb[gr][nt][h] = movmatrix(w);
                            if (h == (ch & 1))
                                part_p[gr][nt] = __hfma2(*reinterpret_cast<const __half2*>(&w), __half2(kSample, kSample), part_p[gr][nt]);
                            if constexpr (SPLIT) {
                                const float2 r = pair_to_f2<__half>(w);
                                pb2[gr][nt][h] = movmatrix(f2_to_pair<__half>(pv[2 * h] - r.x, pv[2 * h + 1] - r.y));
                            }
                        }
                    }
                }
                // outputs
#pragma unroll
                for (uint32_t gr = 0; gr < NG; ++gr) {
                    uint32_t w[4];
                    ldsm4_trans(base + S::data + ch * 8 * D + ((gr * 2 + (lane >> 4)) ^ sw) * 16, w);
                    uint32_t hi[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) hi[i] = __byte_perm(w[i], 0u, 0x4341);
                    auto word = [&](auto j_tag) {
                        constexpr int J = decltype(j_tag)::value;
                        const uint32_t a0 = value_bits<J>(w[0], hi[0]), a1 = value_bits<J>(w[2], hi[2]),
                                       a2 = value_bits<J>(w[1], hi[1]), a3 = value_bits<J>(w[3], hi[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma_f16(o[gr][J][nt], a0, a1, a2, a3, pb[gr][nt][0], pb[gr][nt][1]);
                            if constexpr (SPLIT) mma_f16(o[gr][J][nt], a0, a1, a2, a3, pb2[gr][nt][0], pb2[gr][nt][1]);
                        }
                    };
                    word(std::integral_constant<int, 0>());
                    word(std::integral_constant<int, 1>());
                    word(std::integral_constant<int, 2>());
                    word(std::integral_constant<int, 3>());
                }
            }
        };

        // Takes 8 steps a nibble out of the run's sums, by twice the sample, and the first time half as much again: every
        // run's sums then start about as far below their centre as they end above it.  The sample need not be exact, nor
        // does it follow what a new maximum rescales: what leaves the sums enters zs.
        auto centre = [&](float steps) {
#pragma unroll
            for (uint32_t gr = 0; gr < NG; ++gr) {
                const float back = __uint_as_float((254u << 23) - __float_as_uint(ref[gr])) * (0.25f / kSample);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    __half2 v = part_p[gr][nt];
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) v = __hadd2(v, __shfl_xor_sync(0xffffffffu, v, off));
                    const float2 now = __half22float2(v);
                    part_p[gr][nt] = __half2(0.f, 0.f);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float out = steps * (x ? now.y : now.x);
                        zs[nt][x][gr] = fmaf(out, back, zs[nt][x][gr]);  // (an eighth in each of the lanes that are added up)
                        const float even = out * (2.f / kSample / 16777216.f), odd = 17.f * even;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            o[gr][j][nt][x] -= (j & 1) ? odd : even;
                            o[gr][j][nt][2 + x] -= (j & 1) ? odd : even;
                        }
                    }
                }
            }
        };
        for (uint32_t c = wc0; c < wc1; ++c) {
            __syncwarp();
            load();
            cp_async_wait<STAGES - 1>();
            __syncwarp();
            if ((valid >> (STAGES - 1)) & 1) {
                if ((int)(c * CHUNK + CHUNK) <= least)
                    step(c, slot, std::true_type());
                else
                    step(c, slot, std::false_type());
            } else if (score_at) {  // no such page: nothing of this chunk is seen
                const uint32_t rows = min(ROWS, a.row_pad - block * ROWS);
                for (uint32_t i = lane; i < CHUNK * rows && c * CHUNK + i / rows < sh.vis; i += 32)
                    score_at[((int64_t)(i / rows) - g) * a.row_pad + (int64_t)(i % rows) - 2 * tig] = -INFINITY;
            }
            if ((c - wc0) % (kRun / CH) == kRun / CH - 1) centre(c - wc0 < kRun / CH ? 12.f : 8.f);
            if (score_at) score_at += CHUNK * a.row_pad;
            if (++slot == STAGES) slot = 0;
        }
        // the next piece's rows and first chunks, behind this one's join (which needs the ring itself where shared memory
        // has no room for both)
        const uint32_t next_unit = unit + (cur.c1 - cur.c0);
        if (S::early && next_unit < end) {
            __syncwarp();  // the first load takes the slot of the last chunk, which every lane has read
            cur = piece_at(next_unit);
            if (NT == 1) fetch_rows(cur);  // (more rows would not fit beside the sums)
            slot = lslot;
            begin_loads(cur);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (uint32_t gr = 0; gr < NG; ++gr)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[gr][1][nt][i] -= o[gr][0][nt][i];  // nibbles 1 and 3 from their bytes
                    o[gr][3][nt][i] -= o[gr][2][nt][i];
                }

        // the warps' sums become the block's
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], off);
#pragma unroll
                    for (uint32_t gr = 0; gr < NG; ++gr)
                        zs[nt][x][gr] += __shfl_xor_sync(0xffffffffu, zs[nt][x][gr], off);
                }
                if (!((seen >> (nt * 2 + x)) & 1)) m[nt][x] = -INFINITY;
                if (g == 0) warp_ml[warp][nt * 8 + 2 * tig + x] = make_float2(m[nt][x], l[nt][x]);
            }
        if (!S::early) cp_async_wait<0>();
        __syncthreads();  // every warp is through its chunks, its maxima and sums are there
        const uint32_t seg = unit == begin ? 0 : 1;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt > 0) __syncthreads();
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t r = nt * 8 + 2 * tig + x;
                float top = -INFINITY;
#pragma unroll
                for (uint32_t v = 0; v < kWarps; ++v) top = fmaxf(top, warp_ml[v][r].x);
                // a warp that saw nothing has l = 0, or a NaN that has to stay
                const float f = m[nt][x] == -INFINITY ? l[nt][x] : m[nt][x] == top ? 1.f : ex2(m[nt][x] - top);
                float* at = merge + (warp * 8 + 2 * tig + x) * S::pitch + 4 * g;
#pragma unroll
                for (uint32_t gr = 0; gr < NG; ++gr) {
                    // the group's power of two (exactly inverted), and 2^24 or 2^20 of the nibble
                    const float back = __uint_as_float((254u << 23) - __float_as_uint(ref[gr])) * 1048576.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int cb = 0; cb < 2; ++cb)
                            at[gr * 64 + cb * 32 + j] =
                                fmaf(o[gr][j][nt][cb * 2 + x], (j & 1) ? back : back * 16.f, zs[nt][x][gr]) * f;
                }
            }
            __syncthreads();
#pragma unroll
            for (uint32_t r8 = warp; r8 < 8; r8 += kWarps) {
                const uint32_t r = nt * 8 + r8, row = block * ROWS + r;
                if (row >= all_rows) continue;
                float top = -INFINITY, sum = 0.f;
#pragma unroll
                for (uint32_t v = 0; v < kWarps; ++v) top = fmaxf(top, warp_ml[v][r].x);
#pragma unroll
                for (uint32_t v = 0; v < kWarps; ++v) {
                    const float2 ml = warp_ml[v][r];
                    sum += ml.x == -INFINITY || ml.x == top ? ml.y : ml.y * ex2(ml.x - top);
                }
                const uint32_t qi = row / a.group, qh = head * a.group + row % a.group;
                T* dst = static_cast<T*>(a.out) + ((uint64_t)(sh.start + qi) * a.heads + qh) * D;
                const uint64_t slot_at = (uint64_t)(2 * blockIdx.x + seg) * ROWS + r;
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
                for (uint32_t ch = lane * 2; ch < D; ch += 64) {
                    float2 v = make_float2(0.f, 0.f);
#pragma unroll
                    for (uint32_t w = 0; w < kWarps; ++w) {
                        const float2 t = *reinterpret_cast<const float2*>(merge + (w * 8 + r8) * S::pitch + ch);
                        v.x += t.x;
                        v.y += t.y;
                    }
                    if (whole)
                        *reinterpret_cast<uint32_t*>(dst + ch) = f2_to_pair<T>(v.x * inv, v.y * inv);
                    else
                        *reinterpret_cast<float2*>(a.part_o + slot_at * D + ch) = v;
                }
                if (lane == 0) {
                    if (!whole)
                        a.part_ml[slot_at] = make_float2(top, sum);
                    else if (a.scores)
                        a.stats[((uint64_t)b * a.c.kv_heads + head) * a.row_pad + row] = make_float2(top, sum);
                }
            }
        }
        if (next_unit >= end) break;
        unit = next_unit;
        if (!S::early) {
            __syncthreads();
            cur = piece_at(unit);
            slot = lslot;
            begin_loads(cur);
        }
        if (!S::early || NT > 1) fetch_rows(cur);
    }
    cp_async_wait<0>();
}

// Pieces of an item that blocks left in the workspace: slots of blocks `first` .. `last`.
struct Pieces {
    uint32_t first, last, first_slot;
    __device__ __forceinline__ Pieces(const Split& split, uint32_t unit0, uint32_t chunks)
    {
        first = split.block_of(unit0);
        last = split.block_of(unit0 + chunks - 1);
        first_slot = 2 * first + (unit0 == split.begin(first) ? 0 : 1);
    }
    __device__ __forceinline__ uint32_t count() const { return last - first + 1; }
    __device__ __forceinline__ uint32_t slot(uint32_t i) const { return i == 0 ? first_slot : 2 * (first + i); }
};

constexpr uint32_t kJoinThreads = 256;
constexpr uint32_t kJoinGroup = 4;  // warps that join one row, where there are few

// Joins one row of an item from its pieces, GROUP warps together (all of them call it); the first of them stores it.
template <typename T, int D, uint32_t GROUP>
__device__ __forceinline__ void join_row(const AttnParams& a, const Pieces& p, uint32_t rows_per_item, uint32_t r, T* dst,
                                         float2 (*part)[D / 2], float* part_l)
{
    constexpr uint32_t V = D / 64;  // pairs of channels a lane holds
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31, in_group = warp % GROUP, group = warp / GROUP;
    const uint32_t count = p.count();
    float top = -INFINITY;
    for (uint32_t i = lane; i < count; i += 32)
        top = fmaxf(top, a.part_ml[(uint64_t)p.slot(i) * rows_per_item + r].x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    float2 o[V] = {};
    float sum = 0.f;
    // this warp's pieces: every GROUP-th
    for (uint32_t i0 = in_group; i0 < count; i0 += 32 * GROUP) {
        float f = 0.f;
        const uint32_t i_lane = i0 + lane * GROUP;
        if (i_lane < count) {
            const float2 ml = a.part_ml[(uint64_t)p.slot(i_lane) * rows_per_item + r];
            f = ml.x == -INFINITY ? 0.f : ml.x == top ? 1.f : ex2(ml.x - top);
            sum += ml.x == -INFINITY ? ml.y : ml.y * f;  // a NaN stays
        }
        const uint32_t here = min(32u, (count - i0 + GROUP - 1) / GROUP);
        constexpr uint32_t FLY = V == 4 ? 4 : 8;  // pieces in flight, the last ones too
        for (uint32_t i = 0; i < here; i += FLY) {
            float2 y[FLY][V];
#pragma unroll
            for (uint32_t n = 0; n < FLY; ++n) {
                const uint32_t k = min(i + n, here - 1);
                const float* src = a.part_o + ((uint64_t)p.slot(i0 + k * GROUP) * rows_per_item + r) * D;
#pragma unroll
                for (uint32_t v = 0; v < V; ++v) y[n][v] = *reinterpret_cast<const float2*>(src + v * 64 + lane * 2);
            }
#pragma unroll
            for (uint32_t n = 0; n < FLY; ++n) {
                const float fi = i + n < here ? __shfl_sync(0xffffffffu, f, (i + n) & 31) : 0.f;
                if (i + n < here) {
#pragma unroll
                    for (uint32_t v = 0; v < V; ++v) {
                        o[v].x = fmaf(y[n][v].x, fi, o[v].x);
                        o[v].y = fmaf(y[n][v].y, fi, o[v].y);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if constexpr (GROUP > 1) {
        named_bar_sync(1 + group, GROUP * 32);  // (the last row's sums are read)
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) part[warp][v * 32 + lane] = o[v];
        if (lane == 0) part_l[warp] = sum;
        named_bar_sync(1 + group, GROUP * 32);
        if (in_group != 0) return;
#pragma unroll
        for (uint32_t w = 1; w < GROUP; ++w) {
            sum += part_l[warp + w];
#pragma unroll
            for (uint32_t v = 0; v < V; ++v) {
                const float2 y = part[warp + w][v * 32 + lane];
                o[v].x += y.x;
                o[v].y += y.y;
            }
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (uint32_t v = 0; v < V; ++v)
        *reinterpret_cast<uint32_t*>(dst + v * 64 + lane * 2) = f2_to_pair<T>(o[v].x * inv, o[v].y * inv);
}

// The first join_blocks blocks join the items that lie in several blocks' shares; the others add up the weights, each of an
// equal piece of all positions, from the scores.  With few query rows (`by_rows`) every row looks for its own item, four
// warps a row.  With many, a warp a row, every boundary between two shares stands for the item it cuts, if it is the first to do so:
// there are at most as many such items as blocks, and they are found in shared memory alone.  What depends on the call's
// inputs is worked out before the wait for the first kernel, which has waited for the inputs itself.
// With weights, the kernel does not let its dependents start early: blocks of the next attention that come into registers
// freed piecemeal leave holes that its last ones do not fit (they then ran after the others: 48 x 8192 tokens 128 us, not
// 100).
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads, 3) kv4_join_kernel(AttnParams a, uint32_t rows_per_item, uint32_t grid1,
                                                                   uint32_t join_blocks, bool by_rows)
{
    constexpr uint32_t WARPS = kJoinThreads / 32;
    extern __shared__ uint32_t ustart[];  // [batch + 1], then the chunks of a sequence's items [batch]
    __shared__ float2 row_ml[kJoinThreads];
    __shared__ float2 part[WARPS][D / 2];
    __shared__ float part_l[WARPS];
    __shared__ uint32_t scan_part[WARPS];
    const uint32_t* seq_chunks = ustart + a.s.batch + 1;
    const uint32_t tid = threadIdx.x, warp = tid / 32;
    lay_out<kJoinThreads>(a, rows_per_item, ustart, scan_part, ustart + a.s.batch + 1);
    const uint32_t total = ustart[a.s.batch];
    if (total == 0) {
        griddep_wait();
        return;
    }
    const Split split(total, grid1, a.chunk, a.items);
    if (blockIdx.x < join_blocks) {
        bool waited = false;
        auto wait = [&]() {
            if (waited) return;
            waited = true;
            griddep_wait();
            if (!a.scores) griddep_launch_dependents();
        };
        const uint32_t most_rows = min(rows_per_item, a.group * a.max_queries);
        const uint64_t units = by_rows ? (uint64_t)a.s.tokens * a.heads : (uint64_t)(split.blocks - 1) * most_rows;
        const uint32_t group = by_rows ? kJoinGroup : 1, groups = WARPS / group;
        for (uint64_t x = blockIdx.x * groups + warp / group; x < units; x += join_blocks * groups) {
            uint32_t b, head, row, unit0;  // sequence, key head, row of its rows, the item's first chunk on the line
            SeqShape sh;
            if (by_rows) {
                const uint32_t token = (uint32_t)(x / a.heads), qh = (uint32_t)(x % a.heads);
                uint32_t hi = a.s.batch;
                b = 0;
                while (b < hi) {
                    const uint32_t mid = (b + hi) / 2;
                    if (__ldg(a.s.token_start + mid + 1) <= (int32_t)token)
                        b = mid + 1;
                    else
                        hi = mid;
                }
                if (b == a.s.batch) continue;
                sh = seq_shape(a, b, rows_per_item);
                if (token < sh.start || token - sh.start >= sh.queries) continue;
                head = qh / a.group;
                row = (token - sh.start) * a.group + qh % a.group;
                unit0 = ustart[b] + (head * sh.blocks + row / rows_per_item) * sh.chunks;
            } else {
                const uint32_t at = (uint32_t)(x / most_rows), cut = split.begin(at + 1);
                b = seq_of(ustart, a.s.batch, cut);
                const uint32_t item = (cut - ustart[b]) / seq_chunks[b];
                unit0 = ustart[b] + item * seq_chunks[b];
                if (unit0 == cut || split.block_of(unit0) != at) continue;  // cuts no item, or not as the first
                sh = seq_shape(a, b, rows_per_item);
                head = item / sh.blocks;
                row = item % sh.blocks * rows_per_item + (uint32_t)(x % most_rows);
                if (row >= sh.queries * a.group) continue;
            }
            const Pieces p(split, unit0, sh.chunks);
            if (p.first == p.last) continue;  // written whole
            wait();
            T* dst = static_cast<T*>(a.out) +
                     ((uint64_t)(sh.start + row / a.group) * a.heads + head * a.group + row % a.group) * D;
            if (by_rows)
                join_row<T, D, kJoinGroup>(a, p, rows_per_item, row % rows_per_item, dst, part, part_l);
            else
                join_row<T, D, 1>(a, p, rows_per_item, row % rows_per_item, dst, part, part_l);
        }
        wait();
        return;
    }
    // weights: the line again; a head's row blocks make one run of blocks * chunks units, over which its positions
    // are spread evenly
    const uint32_t wb = blockIdx.x - join_blocks, wblocks = gridDim.x - join_blocks;
    const uint32_t begin = (uint32_t)((uint64_t)total * wb / wblocks), end = (uint32_t)((uint64_t)total * (wb + 1) / wblocks);
    uint32_t unit = begin, b = seq_of(ustart, a.s.batch, unit);
    griddep_wait();
    while (unit < end) {
        while (ustart[b + 1] <= unit) ++b;
        const SeqShape sh = seq_shape(a, b, rows_per_item);
        const uint32_t in_seq = unit - ustart[b];
        const uint32_t run = sh.blocks * sh.chunks, head = in_seq / run, u0 = in_seq % run, u1 = min(run, u0 + (end - unit));
        const uint32_t p0 = (uint32_t)((uint64_t)sh.vis * u0 / run), p1 = (uint32_t)((uint64_t)sh.vis * u1 / run);
        const uint32_t all_rows = sh.queries * a.group;
        const float* scores = a.scores + ((uint64_t)b * a.c.kv_heads + head) * kv4_cap(a.c, a.s) * a.row_pad;
        const int32_t* table = a.s.page_table + (uint64_t)b * a.s.max_pages;
        for (uint32_t r0 = 0; r0 < all_rows; r0 += kJoinThreads) {
            const uint32_t rows = min(kJoinThreads, all_rows - r0);
            __syncthreads();
            // eight lanes a row gather its maximum and sum
            for (uint32_t i = tid / 8; i < (rows + 3) / 4 * 4; i += kJoinThreads / 8) {
                const uint32_t row = min(r0 + i, all_rows - 1), r = row % rows_per_item, l8 = tid & 7;
                const uint32_t lanes = 0xffu << (tid & 24);
                const Pieces p(split, ustart[b] + (head * sh.blocks + row / rows_per_item) * sh.chunks, sh.chunks);
                const uint32_t count = p.count();
                float2 ml = make_float2(-INFINITY, 0.f);
                if (count == 1) {
                    ml = a.stats[((uint64_t)b * a.c.kv_heads + head) * a.row_pad + row];
                } else {
                    for (uint32_t k = l8; k < count; k += 8)
                        ml.x = fmaxf(ml.x, a.part_ml[(uint64_t)p.slot(k) * rows_per_item + r].x);
#pragma unroll
                    for (int off = 4; off > 0; off >>= 1) ml.x = fmaxf(ml.x, __shfl_xor_sync(lanes, ml.x, off));
                    for (uint32_t k = l8; k < count; k += 8) {
                        const float2 x = a.part_ml[(uint64_t)p.slot(k) * rows_per_item + r];
                        ml.y += x.x == -INFINITY || x.x == ml.x ? x.y : x.y * ex2(x.x - ml.x);
                    }
#pragma unroll
                    for (int off = 4; off > 0; off >>= 1) ml.y += __shfl_xor_sync(lanes, ml.y, off);
                }
                if (l8 == 0 && i < kJoinThreads)
                    row_ml[i] = i < rows ? make_float2(ml.x == -INFINITY ? 0.f : ml.x, ml.y == 0.f ? 0.f : 1.f / ml.y)
                                         : make_float2(0.f, 0.f);
            }
            __syncthreads();
            auto add = [&](auto quads_tag) {  // quads_tag: groups of four rows held in registers, 0: any number
                constexpr uint32_t QUADS = decltype(quads_tag)::value, FLY = QUADS == 1 ? 4 : QUADS == 2 ? 2 : 1;
                float2 ml[QUADS ? QUADS * 4 : 1];
#pragma unroll
                for (uint32_t r = 0; r < QUADS * 4; ++r) ml[r] = row_ml[r];
                for (uint32_t t0 = p0 + tid; t0 < p1; t0 += FLY * kJoinThreads) {
                    int64_t at[FLY];
                    float sum[FLY];
                    float4 sv[FLY][QUADS ? QUADS : 1];
#pragma unroll
                    for (uint32_t n = 0; n < FLY; ++n) {
                        const uint32_t t = t0 + n * kJoinThreads;
                        at[n] = t < p1 ? kv4_row(a.c, table, t, head) : -1;
#pragma unroll
                        for (uint32_t q = 0; q < QUADS; ++q)
                            if (t < p1) sv[n][q] = reinterpret_cast<const float4*>(scores + (uint64_t)t * a.row_pad + r0)[q];
                    }
#pragma unroll
                    for (uint32_t n = 0; n < FLY; ++n) sum[n] = at[n] >= 0 ? a.c.weight[at[n]] : 0.f;
#pragma unroll
                    for (uint32_t n = 0; n < FLY; ++n) {
                        float more = 0.f;
                        auto quad = [&](const float4& s4, const float2* m4) {  // (rows that are not there have a factor of 0)
                            more = fmaf(ex2(s4.x - m4[0].x), m4[0].y, more);
                            more = fmaf(ex2(s4.y - m4[1].x), m4[1].y, more);
                            more = fmaf(ex2(s4.z - m4[2].x), m4[2].y, more);
                            more = fmaf(ex2(s4.w - m4[3].x), m4[3].y, more);
                        };
                        if constexpr (QUADS > 0) {
#pragma unroll
                            for (uint32_t q = 0; q < QUADS; ++q) quad(sv[n][q], ml + 4 * q);
                        } else if (at[n] >= 0) {
                            const float4* sp = reinterpret_cast<const float4*>(scores + (uint64_t)t0 * a.row_pad + r0);
                            for (uint32_t q = 0; q * 4 < rows; ++q) quad(sp[q], row_ml + 4 * q);
                        }
                        if (at[n] >= 0) a.c.weight[at[n]] = sum[n] + more;
                    }
                }
            };
            if (rows <= 4)
                add(std::integral_constant<uint32_t, 1>());
            else if (rows <= 8)
                add(std::integral_constant<uint32_t, 2>());
            else
                add(std::integral_constant<uint32_t, 0>());
        }
        unit += u1 - u0;
    }
}

struct AttnWs {
    size_t stats, part_o, part_ml, scores, bytes;
};
// Tiles of 8 rows a block takes.  Blocks of 4 tiles read the cache once for 32 rows, but their sums leave the registers
// and their code the instruction cache: 72 us for 32 rows of 128 channels at 4 x 40000 tokens, two blocks of 2 tiles 63,
// and 52 against 40 at 16 x 4000.
uint32_t tiles_of(uint32_t rows) { return rows <= 8 ? 1 : 2; }

// Queries of a sequence that one pair of launches takes.  With weights, their scores over the whole table have to fit
// kScoreBytes (one query's have room in any case): a prompt of 8192 tokens, 32 heads over 8, would ask for 8.6 GB of them.
// And a launch counts its chunks of 16 tokens, over all key heads and blocks of at least 8 rows, in 32 bits.  0: not even
// one query's.
constexpr uint64_t kScoreBytes = 256ull << 20;
uint32_t queries_of(uint32_t batch, uint32_t heads, uint32_t kv_heads, uint32_t max_queries, uint32_t max_len, bool accumulate)
{
    const uint64_t group = heads / kv_heads, per_row = (uint64_t)batch * kv_heads * max_len * 4;
    const uint64_t chunks = (uint64_t)batch * kv_heads * (max_len / 16 + 1);
    uint64_t n = max_queries;
    if (accumulate && per_row > 0) n = std::min(n, std::max<uint64_t>(1, kScoreBytes / per_row / 4 * 4 / group));
    if (chunks > 0) {
        const uint64_t blocks = UINT32_MAX / chunks;  // rows / 8 + 1 of them
        if (blocks <= group / 8) return 0;
        n = std::min(n, ((blocks - 1) * 8 + 7) / group);
    }
    if (n < max_queries && n * group >= 16) n = std::max<uint64_t>(1, n * group / 16 * 16 / group);  // whole blocks of rows
    return (uint32_t)n;
}

AttnWs layout(uint32_t batch, uint32_t heads, uint32_t kv_heads, uint32_t dim, uint32_t max_queries, uint32_t max_len,
              bool accumulate, uint32_t num_sms)
{
    const uint64_t rows = (uint64_t)(heads / kv_heads) * queries_of(batch, heads, kv_heads, max_queries, max_len, accumulate);
    const uint64_t pad = (rows + 3) / 4 * 4;
    const uint64_t slots = 2ull * num_sms * kMaxBlocks * 8 * tiles_of((uint32_t)std::min<uint64_t>(rows, 1u << 20));
    AttnWs w;
    size_t at = 0;
    auto take = [&](uint64_t n) {
        const size_t here = at;
        at += (n + 255) / 256 * 256;
        return here;
    };
    w.part_ml = take(slots * 8);
    w.part_o = take(slots * dim * 4);
    w.stats = take(accumulate ? (uint64_t)batch * kv_heads * pad * 8 : 0);
    w.scores = take(accumulate ? (uint64_t)batch * kv_heads * max_len * pad * 4 : 0);
    w.bytes = at;
    return w;
}

template <typename T, int D, int NT, int CH>
cudaError_t run(AttnParams& p, bool accumulate, uint32_t num_sms, cudaStream_t st)
{
    using S = AttnSmem<D, NT, CH>;
    static_assert(attn_blocks<D, NT, CH>() <= kMaxBlocks, "workspace too small");
    p.chunk = 16 * CH;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(kv4_attention_kernel<T, D, NT, CH>, S::fixed + (kMaxAttnBatch + 1) * 4, done);
    if (e != cudaSuccess) return e;
    // no more blocks than the page tables have room for chunks
    const uint64_t items = (uint64_t)p.s.batch * p.c.kv_heads * ((p.group * p.max_queries + 8 * NT - 1) / (8 * NT));
    p.items = (uint32_t)std::min<uint64_t>(items, UINT32_MAX);
    const uint64_t most = std::max(items, items * ((uint64_t)p.s.max_pages * p.c.page_size + p.chunk) / kMinTokens + 1);
    const uint32_t grid = (uint32_t)std::min<uint64_t>(most, num_sms * attn_blocks<D, NT, CH>());
    const uint32_t line = (p.s.batch + 1) * 4;
    // The second kernel is one wave of three blocks an SM, with weights one for the rows and two for the weights (a block
    // takes a few microseconds to its first row; four waves of them took 36 us where one takes 20).  Few rows look for
    // their items themselves, many are found by the cuts.  Where the two meet depends on the pieces a row has: lengths up to
    // 4000, 32 heads over 8 of 128 channels, 128 rows 15.3 us, by cuts 16.6, 384 rows 22.0 and 22.0, 576 rows 26.6 and 26.2,
    // 2048 rows 72 and 59; 40000 tokens, 4 queries, 512 rows 62.6 and 67.2, 640 rows 61.4 and 65.9 (64 channels), 1024 rows
    // of one query 108 and 106.
    const uint64_t all_rows = (uint64_t)p.s.tokens * p.heads;
    const bool by_rows = all_rows <= 4 * num_sms;
    const uint32_t groups = kJoinThreads / 32 / (by_rows ? kJoinGroup : 1);
    const uint64_t rows = by_rows ? all_rows : (uint64_t)(grid - 1) * std::min(8u * NT, p.group * p.max_queries);
    const uint32_t weights = accumulate ? (uint32_t)std::min<uint64_t>(most, 2 * num_sms) : 0;
    const uint32_t join = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>((rows + groups - 1) / groups, (accumulate ? 1 : 3) * num_sms));
    for (p.first_query = 0; e == cudaSuccess && p.first_query < p.all_queries; p.first_query += p.max_queries) {
        e = launch_pdl(kv4_attention_kernel<T, D, NT, CH>, dim3(grid), dim3(S::warps * 32), S::fixed + line, st, p);
        if (e == cudaSuccess)
            e = launch_pdl(kv4_join_kernel<T, D>, dim3(join + weights), dim3(kJoinThreads), line + p.s.batch * 4, st, p,
                           8u * NT, grid, join, by_rows);
    }
    return e;
}

template <typename T, int D>
cudaError_t run_dim(AttnParams& p, bool accumulate, uint32_t num_sms, cudaStream_t st)
{
    if (tiles_of(std::min(p.group * p.max_queries, 1u << 20)) == 2) return run<T, D, 2, 1>(p, accumulate, num_sms, st);
    // chunks of 32 tokens, where pages hold whole ones: half the steps, and two chains of products to overlap
    if constexpr (D < 256)
        if (p.c.page_size % 32 == 0) return run<T, D, 1, 2>(p, accumulate, num_sms, st);
    return run<T, D, 1, 1>(p, accumulate, num_sms, st);
}

}  // namespace

bool kv4_attention_fits(uint32_t batch, uint32_t heads, uint32_t kv_heads, uint32_t max_queries, uint32_t max_len,
                        bool accumulate)
{
    return max_queries == 0 || queries_of(batch, heads, kv_heads, max_queries, max_len, accumulate) > 0;
}

size_t kv4_attention_workspace(uint32_t batch, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                               uint32_t max_queries, uint32_t max_len, bool accumulate, uint32_t num_sms)
{
    return layout(batch, heads, kv_heads, head_dim, max_queries, max_len, accumulate, num_sms).bytes;
}

cudaError_t launch_kv4_attention(const Kv4Attention& a, void* workspace, uint32_t num_sms, cudaStream_t st)
{
    const uint32_t cap = a.seqs.max_pages * a.cache.page_size;
    const AttnWs w = layout(a.seqs.batch, a.heads, a.cache.kv_heads, a.cache.head_dim, a.max_queries, cap, a.accumulate,
                            num_sms);
    uint8_t* base = static_cast<uint8_t*>(workspace);
    AttnParams p{};
    p.c = a.cache;
    p.s = a.seqs;
    p.q = a.q;
    p.out = a.out;
    p.q_stride = a.q_stride;
    p.heads = a.heads;
    p.group = a.heads / a.cache.kv_heads;
    p.all_queries = std::min(a.max_queries, a.seqs.tokens);
    p.max_queries = queries_of(a.seqs.batch, a.heads, a.cache.kv_heads, a.max_queries, cap, a.accumulate);
    p.row_pad = (p.group * p.max_queries + 3) / 4 * 4;
    p.scale = a.scale;
    p.stats = reinterpret_cast<float2*>(base + w.stats);
    p.part_o = reinterpret_cast<float*>(base + w.part_o);
    p.part_ml = reinterpret_cast<float2*>(base + w.part_ml);
    p.scores = a.accumulate ? reinterpret_cast<float*>(base + w.scores) : nullptr;
    switch (a.cache.head_dim) {
        case 64:
            return a.bf16 ? run_dim<__nv_bfloat16, 64>(p, a.accumulate, num_sms, st)
                          : run_dim<__half, 64>(p, a.accumulate, num_sms, st);
        case 128:
            return a.bf16 ? run_dim<__nv_bfloat16, 128>(p, a.accumulate, num_sms, st)
                          : run_dim<__half, 128>(p, a.accumulate, num_sms, st);
        default:
            return a.bf16 ? run_dim<__nv_bfloat16, 256>(p, a.accumulate, num_sms, st)
                          : run_dim<__half, 256>(p, a.accumulate, num_sms, st);
    }
}

}  // namespace b2sq
