// kv4_append.cu — writes new keys and values into the 4-bit paged cache.
//
// Per group of 64 channels (v saturated to fp16's finite range):
//   z = fp16(min v), s = fp16((max v - min v) / 15)
//   q = clamp(rint((v - z) / s), 0, 15), ties to even; s = 0 gives q = 0
// A NaN makes its group's s and z NaN, so it is not lost in the cache.
//
// HBM would bound it (2 bytes a channel in, 0.56 out, 2 more where the cached
// values are asked for) with fewer than 18 instructions a channel at the rate they
// issue here; it takes 28, and the issue slots (75% full) and the wait for a
// block's places in front of its first loads do.  Eight lanes hold a group, one
// 16-byte load and one 4-byte store of nibbles each; extrema in packed 16-bit operations and three shuffles; the
// quotient as a saturated product with 1 / (15 s), whose exact remainder tells
// whether it was rounded right.  Inputs of 8 or 11 significant bits meet the
// border between two steps often, so those lanes decide it exactly, with what
// the difference v - z has beyond fp32.
//
// 7 prompts of up to 4001 tokens, 8 heads of 128 channels: 42 us (173 MB, 4.1
// TB/s); 16 tokens 2.9 us.
#include "kv4.cuh"

#include <algorithm>

namespace b2sq {

namespace {

constexpr uint32_t kAppendThreads = 256;
constexpr uint32_t kAppendTokens = 8;  // tokens of a block at most
constexpr float kHalfMax = 65504.f;
constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, held in the low bits

constexpr uint32_t kRoundBits = 0x3f400000u;  // sum of kRound's bits shifted left by 0, 4, ..., 28

constexpr float kFifteenth = 1.f / 15.f;

__device__ __forceinline__ float approx_rcp(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Smaller and larger of packed pairs; a NaN wins.
template <typename T>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b);
template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t min2<__half>(uint32_t a, uint32_t b)
{
    uint32_t d;
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
template <>
__device__ __forceinline__ uint32_t max2<__half>(uint32_t a, uint32_t b)
{
    uint32_t d;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
template <>
__device__ __forceinline__ uint32_t min2<__nv_bfloat16>(uint32_t a, uint32_t b)
{
    uint32_t d;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
template <>
__device__ __forceinline__ uint32_t max2<__nv_bfloat16>(uint32_t a, uint32_t b)
{
    uint32_t d;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// Eight nibbles whose quotients fp32 sees on a border between two steps or off it: on a border, what rounding x - base
// left out (Knuth's two-sum) decides.  A border has 16 bits, so the rounded difference is on the same side of it as x -
// base, or on it.  The difference of numbers with 11 bits is exact unless one of them is below 2^-12 of it.
template <typename T>
__device__ uint32_t settle_borders(uint32_t packed, const T* x8, float base, float step)
{
#pragma unroll 1
    for (int i = 0; i < 32; i += 4, ++x8) {
        const float x = (float)*x8, f = x - base, b = f - x, rest = (x - (f - b)) + (-base - b);
        const float q = (float)(packed >> i & 15), r2 = 2.f * fmaf(-q, step, f);
        if (r2 == step && rest > 0.f && q < 15.f) packed += 1u << i;
        if (r2 == -step && rest < 0.f && q > 0.f) packed -= 1u << i;
    }
    return packed;
}

// A block takes a run of tokens: finds their places, then quantises their keys and values, eight channels a thread.
template <typename T>
__global__ void __launch_bounds__(kAppendThreads)
    kv4_append_kernel(Kv4Cache c, Kv4Seqs s, const T* __restrict__ k, const T* __restrict__ v, uint64_t k_stride,
                      uint64_t v_stride, T* __restrict__ k_out, T* __restrict__ v_out, uint32_t tokens_each)
{
    __shared__ int64_t place[kAppendTokens];  // cache row of head 0, -1 for a token without a place
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t tid = threadIdx.x, token0 = blockIdx.x * tokens_each;
    const uint32_t here = min(tokens_each, s.tokens - token0);
    if (tid < here) {
        const uint32_t token = token0 + tid;
        // the sequence that holds this token: the last one starting at or before it
        uint32_t lo = 0, hi = s.batch;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (__ldg(s.token_start + mid + 1) <= (int32_t)token)
                lo = mid + 1;
            else
                hi = mid;
        }
        int64_t row = -1;
        if (lo < s.batch) {
            uint32_t start;
            const uint32_t count = kv4_new_rows(s, lo, start);
            // the new tokens are the sequence's last ones; what falls outside the table is not written
            const int64_t p = (int64_t)kv4_len(s, lo) - count + ((int64_t)token - start);
            if (token >= start && token - start < count && p >= 0 && p < (int64_t)kv4_cap(c, s))
                row = kv4_row(c, s.page_table + (uint64_t)lo * s.max_pages, (uint32_t)p, 0);
        }
        place[tid] = row;
    }
    __syncthreads();

    const uint32_t units = c.kv_heads * c.head_dim / 8;  // of keys, and of values
    const uint32_t lane8 = tid & 7, mask = 0xffu << (tid & 24);
    const uint32_t dshift = __ffs(c.head_dim) - 1, gshift = dshift - 6;
    for (uint32_t u = tid; u < 2 * units; u += kAppendThreads) {  // whole groups of eight lanes: units is a multiple of 8
        const bool is_v = u >= units;
        const uint32_t ch = (is_v ? u - units : u) * 8, head = ch >> dshift, in_head = ch & (c.head_dim - 1);
        const uint64_t stride = is_v ? v_stride : k_stride, out_stride = (uint64_t)units * 8;
        const T* src = (is_v ? v : k) + token0 * stride + ch;
        T* out = is_v ? v_out : k_out;
        if (out) out += token0 * out_stride + ch;
        // of head 0's row in the cache: this head's nibbles and group
        uint32_t* data = reinterpret_cast<uint32_t*>(is_v ? c.v : c.k) + ((uint64_t)head * c.page_size << (dshift - 3)) + in_head / 8;
        uint32_t* scale = reinterpret_cast<uint32_t*>(is_v ? c.v_scale : c.k_scale) +
                          ((uint64_t)head * c.page_size << gshift) + in_head / kKv4Group;
        float* weight = !is_v && in_head == 0 && c.weight ? c.weight + (uint64_t)head * c.page_size : nullptr;
        uint4 next = place[0] >= 0 ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
        for (uint32_t t = 0; t < here; ++t) {
            const uint32_t w[4] = {next.x, next.y, next.z, next.w};
            const int64_t row0 = place[t];
            src += stride;
            if (t + 1 < here && place[t + 1] >= 0) next = *reinterpret_cast<const uint4*>(src);
            T* to = out;
            if (out) out += out_stride;
            if (row0 < 0) continue;
            uint32_t lo2 = min2<T>(min2<T>(w[0], w[1]), min2<T>(w[2], w[3]));
            uint32_t hi2 = max2<T>(max2<T>(w[0], w[1]), max2<T>(w[2], w[3]));
#pragma unroll
            for (int off = 4; off > 0; off >>= 1) {
                lo2 = min2<T>(lo2, __shfl_xor_sync(mask, lo2, off));
                hi2 = max2<T>(hi2, __shfl_xor_sync(mask, hi2, off));
            }
            const float2 lo = pair_to_f2<T>(lo2), hi = pair_to_f2<T>(hi2);
            const bool nan = !(lo.x == lo.x && lo.y == lo.y);
            const float mn = fminf(fmaxf(fminf(lo.x, lo.y), -kHalfMax), kHalfMax);
            const float mx = fminf(fmaxf(fmaxf(hi.x, hi.y), -kHalfMax), kHalfMax);
            // (mx - mn) / 15 in fp32: the product with the rounded 1 / 15 and one correction by its exact remainder, which is
            // the rounded quotient (Markstein, IBM J. Res. Dev. 34, 1990)
            const float range = mx - mn, s0 = range * kFifteenth, s1 = fmaf(fmaf(-s0, 15.f, range), kFifteenth, s0);
            const __half sh = __float2half_rn(s1), zh = __float2half_rn(mn);
            const float step = __half2float(sh), base = __half2float(zh), half_step = 0.5f * step;
            const float inv15 = step > 0.f ? approx_rcp(15.f * step) : 0.f;  // (its errors are mended below)
            float f[8], q[8], worst = 0.f;
            uint32_t packed = 0u - kRoundBits;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 x = pair_to_f2<T>(w[i]);
                f[2 * i] = x.x - base;
                f[2 * i + 1] = x.y - base;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float r = fmaf(__saturatef(f[i] * inv15), 15.f, kRound);
                q[i] = r - kRound;
                worst = fmaxf(worst, fabsf(fmaf(-q[i], step, f[i])));  // of f, the remainder exactly
                packed += __float_as_uint(r) << (4 * i);
            }
            if (worst >= half_step && step > 0.f) {  // a border, a quotient rounded wrong, or a value that saturates
                packed = 0;
                bool border = false;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float r2 = 2.f * fmaf(-q[i], step, f[i]);
                    const bool odd = ((int)q[i] & 1) != 0;
                    if (r2 > step || (r2 == step && odd)) q[i] = fminf(q[i] + 1.f, 15.f);
                    if (r2 < -step || (r2 == -step && odd)) q[i] = fmaxf(q[i] - 1.f, 0.f);
                    border |= fabsf(r2) == step;
                    packed |= (uint32_t)q[i] << (4 * i);
                }
                if (border) {  // (on one, with ordinary numbers, in a warp of twenty)
                    bool cut = false;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        cut |= fminf(fabsf(f[i] + base), fabsf(base)) < f[i] * (1.f / 4096.f);
                    if (cut && base != 0.f) {
                        packed = settle_borders(packed, src - stride, base, step);
#pragma unroll
                        for (int i = 0; i < 8; ++i) q[i] = (float)(packed >> (4 * i) & 15);
                    }
                }
            }
            data[row0 << (dshift - 3)] = packed;
            if (lane8 == 0) {
                scale[row0 << gshift] =
                    nan ? 0x7fff7fffu : (uint32_t)__half_as_ushort(sh) | ((uint32_t)__half_as_ushort(zh) << 16);
                if (weight) weight[row0] = 0.f;
            }
            if (to) {
                const float b0 = nan ? __int_as_float(0x7fffffff) : base;
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[i] = f2_to_pair<T>(fmaf(q[2 * i], step, b0), fmaf(q[2 * i + 1], step, b0));
                *reinterpret_cast<uint4*>(to) = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
    }
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4Cache& c, const Kv4Seqs& s, const void* k, const void* v, bool bf16,
                              uint64_t k_stride, uint64_t v_stride, void* k_out, void* v_out, uint32_t num_sms,
                              cudaStream_t st)
{
    // a token a block until every SM has several, then runs of them
    const uint32_t each = std::max(1u, std::min(kAppendTokens, s.tokens / (8 * num_sms)));
    const dim3 grid((s.tokens + each - 1) / each);
    if (bf16)
        return launch_pdl(kv4_append_kernel<__nv_bfloat16>, grid, dim3(kAppendThreads), 0, st, c, s,
                          static_cast<const __nv_bfloat16*>(k), static_cast<const __nv_bfloat16*>(v), k_stride,
                          v_stride, static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out), each);
    return launch_pdl(kv4_append_kernel<__half>, grid, dim3(kAppendThreads), 0, st, c, s,
                      static_cast<const __half*>(k), static_cast<const __half*>(v), k_stride, v_stride,
                      static_cast<__half*>(k_out), static_cast<__half*>(v_out), each);
}

}  // namespace b2sq
