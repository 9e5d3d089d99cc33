// kv4_evict.cu — thins sequences of the 4-bit cache out to a budget of tokens.
//
// A sequence of n > budget tokens keeps, in every head by itself, its newest
// `recent` tokens and of the others the budget - recent with the largest
// accumulated attention weight (equal weights: the lower position; a NaN
// counts as the largest).  Kept tokens stay in order and are copied, with
// their weights, to the pages of a second table; shorter sequences are copied
// whole.
//
// The threshold is found by a radix search over the weights' sortable bits
// (four passes of 8 bits over keys in shared memory, of long sequences as many
// as fit: 1 x 60785 tokens, one head, 130 us, with none of them 245), places by
// prefix sums within and over the warps.  Every block of a head repeats that search
// and copies its own share of the kept rows, so no block waits for another.
//
// The copy is bound by HBM, the search by the latency of its passes: 32 x 8192
// tokens, 8 heads of 128 channels, down to 2048: 51 us (159 MB, 3.1 TB/s);
// 1 x 1040 down to 1024: 7.4 us.
#include "kv4.cuh"

#include <algorithm>
#include <atomic>

namespace b2sq {

namespace {

constexpr uint32_t kEvictThreads = 512;
constexpr uint32_t kEvictWarps = kEvictThreads / 32;
constexpr uint32_t kEvictKeys = 40960;  // keys held in shared memory (160 KB); longer sequences re-read the others
constexpr uint32_t kEvictRows = 2048;   // kept rows one block lists at a time
constexpr uint32_t kEvictFly = 4;       // copies of a thread in flight

// Bits that order as the weights do; -0 equals +0, NaN is above infinity.
__device__ __forceinline__ uint32_t weight_key(float w)
{
    if (w != w) return 0xffffffffu;
    const uint32_t b = __float_as_uint(w + 0.f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

template <uint32_t NG>
struct ScaleWord;  // a row's steps and bases of its keys, or values
template <>
struct ScaleWord<1> {
    using type = uint32_t;
};
template <>
struct ScaleWord<2> {
    using type = uint2;
};
template <>
struct ScaleWord<4> {
    using type = uint4;
};

// Rows turn, turn + STEP, ... of `count`: one word of rows of PITCH words each.
template <uint32_t STEP, uint32_t PITCH, typename W>
__device__ __forceinline__ void copy_rows(W* base, const longlong2* at, uint32_t turn, uint32_t count)
{
    for (uint32_t j0 = turn; j0 < count; j0 += kEvictFly * STEP) {
        W v[kEvictFly];
        int64_t to[kEvictFly];
#pragma unroll
        for (uint32_t n = 0; n < kEvictFly; ++n) {
            to[n] = -1;
            if (j0 + n * STEP < count) {
                const longlong2 a = at[j0 + n * STEP];
                to[n] = a.y;
                if (a.y >= 0) v[n] = base[a.x * PITCH];
            }
        }
#pragma unroll
        for (uint32_t n = 0; n < kEvictFly; ++n)
            if (to[n] >= 0) base[to[n] * PITCH] = v[n];
    }
}

template <uint32_t NG>  // groups of 64 channels
__global__ void __launch_bounds__(kEvictThreads, 2)
    kv4_evict_kernel(Kv4Cache c, const int32_t* __restrict__ page_table, uint32_t max_pages,
                     const int32_t* __restrict__ seq_lens, const int32_t* __restrict__ new_table,
                     uint32_t new_max_pages, uint32_t budget, uint32_t recent, int32_t* __restrict__ new_lens,
                     uint32_t key_slots, uint32_t row_slots)
{
    extern __shared__ __align__(16) uint32_t ev_smem[];
    uint32_t* keys = ev_smem;              // [key_slots]
    uint32_t* rows = ev_smem + key_slots;  // [row_slots] positions of kept tokens
    longlong2* at = reinterpret_cast<longlong2*>(rows + row_slots);  // [row_slots] cache rows they come from and go to
    __shared__ uint32_t hist[256];
    __shared__ uint32_t warp_gt[kEvictWarps], warp_eq[kEvictWarps];
    __shared__ uint32_t sel_digit, sel_above;

    griddep_wait();
    griddep_launch_dependents();
    const uint32_t b = blockIdx.z, head = blockIdx.y;
    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const int32_t* table = page_table + (uint64_t)b * max_pages;
    const int32_t* dst_table = new_table + (uint64_t)b * new_max_pages;
    const uint32_t n = min((uint32_t)max(__ldg(seq_lens + b), 0), max_pages * c.page_size);
    const uint32_t kept = min(min(n, budget), new_max_pages * c.page_size);
    if (new_lens && blockIdx.x == 0 && head == 0 && tid == 0) new_lens[b] = (int32_t)kept;
    // this block's share of the kept rows
    const uint32_t d0 = (uint32_t)((uint64_t)kept * blockIdx.x / gridDim.x);
    const uint32_t d1 = (uint32_t)((uint64_t)kept * (blockIdx.x + 1) / gridDim.x);
    if (d0 == d1) return;

    const bool all = n <= kept;
    const uint32_t newest = min(recent, kept);
    const uint32_t old = all ? 0 : n - newest;      // candidates
    const uint32_t want = all ? 0 : kept - newest;  // of them kept

    // keys of positions i .. i + 3 (i a multiple of 4, so they are neighbours on one page); past the candidates: anything
    auto read_keys = [&](uint32_t i, uint32_t (&k)[4]) {
        const int64_t r = i < old ? kv4_row(c, table, i, head) : -1;
        const float4 w = r < 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : __ldg(reinterpret_cast<const float4*>(c.weight + r));
        k[0] = weight_key(w.x), k[1] = weight_key(w.y), k[2] = weight_key(w.z), k[3] = weight_key(w.w);
        if (r < 0) k[0] = k[1] = k[2] = k[3] = 0;
    };
    const uint32_t held = min(old, key_slots);  // (key_slots is a multiple of 4)
    constexpr uint32_t FLY = 2, STRIDE = 4 * kEvictThreads;
    for (uint32_t i0 = tid * 4; i0 < held; i0 += FLY * STRIDE) {
        uint32_t k[FLY][4];
#pragma unroll
        for (uint32_t n = 0; n < FLY; ++n) read_keys(i0 + n * STRIDE, k[n]);
#pragma unroll
        for (uint32_t n = 0; n < FLY; ++n)
            if (i0 + n * STRIDE < held)
                *reinterpret_cast<uint4*>(keys + i0 + n * STRIDE) = make_uint4(k[n][0], k[n][1], k[n][2], k[n][3]);
    }
    auto keys_at = [&](uint32_t i, uint32_t (&k)[4]) {
        if (i < held) {
            const uint4 v = *reinterpret_cast<const uint4*>(keys + i);
            k[0] = v.x, k[1] = v.y, k[2] = v.z, k[3] = v.w;
        } else {
            read_keys(i, k);
        }
    };

    // the want-th largest key: `prefix` gathers its digits, `above` counts larger ones
    uint32_t prefix = 0, above = 0;
    if (want > 0 && want < old) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (uint32_t i = tid; i < 256; i += kEvictThreads) hist[i] = 0;
            __syncthreads();
            auto count = [&](uint32_t i, const uint32_t (&k)[4]) {
#pragma unroll
                for (uint32_t n = 0; n < 4; ++n)
                    if (i + n < old && (shift == 24 || ((k[n] ^ prefix) >> (shift + 8)) == 0))
                        atomicAdd(&hist[(k[n] >> shift) & 255u], 1u);
            };
            uint32_t i = tid * 4;
            for (; i < held; i += STRIDE) {
                uint32_t k[4];
                keys_at(i, k);
                count(i, k);
            }
            for (; i < old; i += FLY * STRIDE) {
                uint32_t k[FLY][4];
#pragma unroll
                for (uint32_t n = 0; n < FLY; ++n) read_keys(i + n * STRIDE, k[n]);
#pragma unroll
                for (uint32_t n = 0; n < FLY; ++n) count(i + n * STRIDE, k[n]);
            }
            __syncthreads();
            if (warp == 0) {
                uint32_t mine[8], sum = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {  // lane l holds digits 255 - 8 l downwards
                    mine[j] = hist[255 - (lane * 8 + j)];
                    sum += mine[j];
                }
                uint32_t incl = sum;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const uint32_t t = __shfl_up_sync(0xffffffffu, incl, off);
                    if (lane >= (uint32_t)off) incl += t;
                }
                uint32_t run = above + incl - sum;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (run < want && run + mine[j] >= want) {
                        sel_digit = 255 - (lane * 8 + j);
                        sel_above = run;
                    }
                    run += mine[j];
                }
            }
            __syncthreads();
            prefix |= sel_digit << shift;
            above = sel_above;
        }
    }
    const uint32_t ties = want - above;  // of the keys equal to `prefix`, the first ones
    const bool take_all_old = want == old, take_none = want == 0;

    // each warp walks a run of positions, four a lane: first its counts, then the places.  Larger ones are counted in
    // the lower half of a word, equal ones in the upper (a run of 128 positions a step, so a step's sums fit).
    const uint32_t run = (old + kEvictWarps * 128 - 1) / (kEvictWarps * 128) * 128;
    const uint32_t w0 = min(warp * run, old), w1 = min(w0 + run, old);
    auto marks = [&](uint32_t i, uint32_t n, uint32_t key) -> uint32_t {  // 1: larger, 1 << 16: equal
        if (i + n >= w1) return 0u;
        if (take_all_old || key > prefix) return 1u;
        return key == prefix ? 1u << 16 : 0u;
    };
    uint32_t gt = 0, eq = 0;
    if (!take_none)
        for (uint32_t i0 = w0 + lane * 4; i0 < w1; i0 += FLY * 128) {
            uint32_t k[FLY][4], both = 0;
#pragma unroll
            for (uint32_t f = 0; f < FLY; ++f) keys_at(i0 + f * 128, k[f]);
#pragma unroll
            for (uint32_t f = 0; f < FLY; ++f)
#pragma unroll
                for (uint32_t n = 0; n < 4; ++n) both += marks(i0 + f * 128, n, k[f][n]);
            gt += both & 0xffffu;
            eq += both >> 16;
        }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        gt += __shfl_xor_sync(0xffffffffu, gt, off);
        eq += __shfl_xor_sync(0xffffffffu, eq, off);
    }
    if (lane == 0) {
        warp_gt[warp] = gt;
        warp_eq[warp] = eq;
    }
    __syncthreads();
    uint32_t gt0 = 0, eq0 = 0;
    for (uint32_t i = 0; i < warp; ++i) {
        gt0 += warp_gt[i];
        eq0 += warp_eq[i];
    }
    // places of the warp's kept tokens
    const uint32_t to0 = gt0 + min(eq0, ties), to1 = gt0 + gt + min(eq0 + eq, ties);

    // a thread copies the same 16-byte piece of every row that is its turn: keys, then values
    constexpr uint32_t PIECES = 4 * NG, ROWS = kEvictThreads / PIECES;
    const uint32_t piece = tid % PIECES, turn = tid / PIECES;
    uint4* const data = reinterpret_cast<uint4*>(piece < PIECES / 2 ? c.k : c.v) + piece % (PIECES / 2);
    using Scale = typename ScaleWord<NG>::type;
    Scale* const scale = static_cast<Scale*>(tid & 1 ? c.v_scale : c.k_scale);
    for (uint32_t r0 = d0; r0 < d1; r0 += row_slots) {
        const uint32_t r1 = min(r0 + row_slots, d1);
        if (to0 < r1 && to1 > r0) {
            uint32_t g = gt0, e = eq0;  // before this step
            uint32_t k[4], next[4];
            keys_at(w0 + lane * 4, k);
            for (uint32_t base = w0; base < w1; base += 128) {
                const uint32_t i = base + lane * 4;
                uint32_t mine[4], sum = 0;
                keys_at(i + 128, next);  // (on their way behind this step's)
#pragma unroll
                for (uint32_t n = 0; n < 4; ++n) {
                    mine[n] = marks(i, n, k[n]);
                    sum += mine[n];
                    k[n] = next[n];
                }
                uint32_t incl = sum;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const uint32_t t = __shfl_up_sync(0xffffffffu, incl, off);
                    if (lane >= (uint32_t)off) incl += t;
                }
                uint32_t lg = g + ((incl - sum) & 0xffffu), le = e + ((incl - sum) >> 16);
#pragma unroll
                for (uint32_t n = 0; n < 4; ++n) {
                    const bool is_gt = mine[n] == 1u, is_eq = mine[n] > 1u;
                    if (is_gt || (is_eq && le < ties)) {
                        const uint32_t to = lg + min(le, ties);
                        if (to >= r0 && to < r1) rows[to - r0] = i + n;
                    }
                    lg += is_gt;
                    le += is_eq;
                }
                const uint32_t all_sum = __shfl_sync(0xffffffffu, incl, 31);
                g += all_sum & 0xffffu;
                e += all_sum >> 16;
            }
        }
        for (uint32_t to = max(r0, want) + tid; to < r1; to += kEvictThreads) rows[to - r0] = all ? to : n - kept + to;
        __syncthreads();
        for (uint32_t j = tid; j < r1 - r0; j += kEvictThreads) {
            const int64_t src = kv4_row(c, table, rows[j], head), dst = kv4_row(c, dst_table, r0 + j, head);
            at[j] = src < 0 || dst < 0 ? make_longlong2(-1, -1) : make_longlong2(src, dst);
            if (src >= 0 && dst >= 0) c.weight[dst] = c.weight[src];
        }
        __syncthreads();
        copy_rows<ROWS, PIECES / 2>(data, at, turn, r1 - r0);
        copy_rows<kEvictThreads / 2, 1>(scale, at, tid / 2, r1 - r0);
        __syncthreads();
    }
}

// New lengths in the place of the old ones, once no block of the eviction reads them any more.
__global__ void kv4_lens_kernel(int32_t* lens, uint32_t batch, uint32_t cap, uint32_t budget)
{
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b < batch) lens[b] = (int32_t)min(min((uint32_t)max(lens[b], 0), cap), budget);
}

}  // namespace

cudaError_t launch_kv4_evict(const Kv4Cache& c, const int32_t* page_table, uint32_t max_pages, const int32_t* seq_lens,
                             const int32_t* new_table, uint32_t new_max_pages, uint32_t batch, uint32_t budget,
                             uint32_t recent, int32_t* new_lens, uint32_t num_sms, cudaStream_t st)
{
    const uint32_t cap = max_pages * c.page_size;
    budget = std::min(budget, std::min(cap, new_max_pages * c.page_size));  // (no more tokens fit either table)
    const uint64_t heads = (uint64_t)batch * c.kv_heads;
    // a block for every SM; each copies at least 64 rows (twice as many took 64 us instead of 54 at 32 x 8192 tokens and
    // 8 heads: the search is repeated)
    const uint32_t key_slots = std::min(cap, kEvictKeys);
    // where two do not fit on one SM, no more than there are SMs (2 x 131000 tokens to 60000, 8 heads: 521 us; 812 with twelve blocks left for a second turn)
    const bool two = (key_slots * 4 + kEvictRows * 20) * 2 <= 225 * 1024;
    const uint32_t split = (uint32_t)std::max<uint64_t>(
        1, std::min<uint64_t>((num_sms + (two ? heads - 1 : 0)) / heads, std::min<uint64_t>(16, (budget + 63) / 64)));
    const uint32_t row_slots = (std::min(kEvictRows, (budget + split - 1) / split + 1) + 3) / 4 * 4;
    const size_t smem = (size_t)key_slots * 4 + (size_t)row_slots * 20;
    const bool in_place = new_lens == seq_lens;
    int32_t* const lens = in_place ? nullptr : new_lens;
    auto launch = [&](auto kernel, std::atomic<uint64_t>& done) {
        cudaError_t e = allow_smem(kernel, kEvictKeys * 4 + kEvictRows * 20, done);
        if (e == cudaSuccess)
            e = launch_pdl(kernel, dim3(split, c.kv_heads, batch), dim3(kEvictThreads), smem, st, c, page_table, max_pages,
                           seq_lens, new_table, new_max_pages, budget, recent, lens, key_slots, row_slots);
        if (e == cudaSuccess && in_place)
            e = launch_pdl(kv4_lens_kernel, dim3((batch + 255) / 256), dim3(256), 0, st, new_lens, batch, cap, budget);
        return e;
    };
    static std::atomic<uint64_t> done[3];
    switch (c.head_dim) {
        case 64: return launch(kv4_evict_kernel<1>, done[0]);
        case 128: return launch(kv4_evict_kernel<2>, done[1]);
        default: return launch(kv4_evict_kernel<4>, done[2]);
    }
}

}  // namespace b2sq
