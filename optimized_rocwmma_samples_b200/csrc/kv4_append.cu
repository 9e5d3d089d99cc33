// kv4_append.cu — writes new keys and values into the 4-bit paged cache.
//
// Per group of 64 channels (v saturated to fp16's finite range):
//   z = fp16(min v), s = fp16((max v - min v) / 15)
//   q = clamp(rint((v - z) / s), 0, 15), ties to even; s = 0 gives q = 0
// A NaN makes its group's s and z NaN, so it is not lost in the cache.
//
// Bound by HBM (2 bytes a channel in, 0.56 out, 2 more where the cached
// values are asked for) as long as the arithmetic stays near ten instructions
// a channel: eight lanes hold a group, one 16-byte load and one 4-byte store of
// nibbles each; extrema in packed 16-bit operations and three shuffles; the
// quotient as a saturated product with 1 / (15 s), whose exact remainder tells
// whether it was rounded right.  Inputs of 8 or 11 significant bits meet the
// border between two steps often, so those lanes decide it exactly.
#include "kv4.cuh"

#include <algorithm>

namespace b2sq {

namespace {

constexpr uint32_t kAppendThreads = 256;
constexpr uint32_t kAppendTokens = 8;  // tokens of a block at most
constexpr float kHalfMax = 65504.f;
constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, held in the low bits

constexpr uint32_t kRoundBits = 0x3f400000u;  // sum of kRound's bits shifted left by 0, 4, ..., 28

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

    const uint32_t ng = c.head_dim / kKv4Group, units = c.kv_heads * c.head_dim / 8;  // of keys, and of values
    const uint32_t lane8 = tid & 7, mask = 0xffu << (tid & 24);
    const uint32_t shift = __ffs(c.head_dim) - 1;
    for (uint32_t t = 0; t < here; ++t) {
        const int64_t row0 = place[t];
        if (row0 < 0) continue;
        const uint64_t token = token0 + t;
        for (uint32_t u = tid; u < 2 * units; u += kAppendThreads) {  // whole groups of eight lanes: units is a multiple of 8
            const bool is_v = u >= units;
            const uint32_t ch = (is_v ? u - units : u) * 8;
            const uint4 raw = *reinterpret_cast<const uint4*>((is_v ? v + token * v_stride : k + token * k_stride) + ch);
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
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
            const __half sh = __float2half_rn((mx - mn) / 15.f), zh = __float2half_rn(mn);
            const float step = __half2float(sh), base = __half2float(zh), half_step = 0.5f * step;
            const float inv15 = step > 0.f ? 1.f / (15.f * step) : 0.f;
            float f[8], q[8], worst = 0.f;
            uint32_t packed = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 x = pair_to_f2<T>(w[i]);
                f[2 * i] = x.x;
                f[2 * i + 1] = x.y;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = f[i] - base;
                const float r = fmaf(__saturatef(d * inv15), 15.f, kRound);
                q[i] = r - kRound;
                worst = fmaxf(worst, fabsf(fmaf(-q[i], step, d)));  // the remainder, exactly
                packed += __float_as_uint(r) << (4 * i);
            }
            packed -= kRoundBits;
            if (worst >= half_step && step > 0.f) {  // a border, a quotient rounded wrong, or a value that saturates
                packed = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float d = f[i] - base, r2 = 2.f * fmaf(-q[i], step, d);
                    const bool odd = ((int)q[i] & 1) != 0;
                    if (r2 > step || (r2 == step && odd)) q[i] = fminf(q[i] + 1.f, 15.f);
                    if (r2 < -step || (r2 == -step && odd)) q[i] = fmaxf(q[i] - 1.f, 0.f);
                    packed |= (uint32_t)q[i] << (4 * i);
                }
            }
            const uint32_t head = ch >> shift, in_head = ch & (c.head_dim - 1);
            const int64_t row = row0 + (int64_t)head * c.page_size;
            reinterpret_cast<uint32_t*>(is_v ? c.v : c.k)[row * (c.head_dim / 8) + in_head / 8] = packed;
            if (lane8 == 0) {
                const uint32_t g = in_head / kKv4Group;
                const uint32_t sz = nan ? 0x7fff7fffu : (uint32_t)__half_as_ushort(sh) | ((uint32_t)__half_as_ushort(zh) << 16);
                reinterpret_cast<uint32_t*>(is_v ? c.v_scale : c.k_scale)[row * ng + g] = sz;
                if (!is_v && g == 0 && c.weight) c.weight[row] = 0.f;
            }
            T* out = is_v ? v_out : k_out;
            if (out) {
                const float b0 = nan ? __int_as_float(0x7fffffff) : base;
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[i] = f2_to_pair<T>(fmaf(q[2 * i], step, b0), fmaf(q[2 * i + 1], step, b0));
                *reinterpret_cast<uint4*>(out + token * c.kv_heads * c.head_dim + ch) = make_uint4(o[0], o[1], o[2], o[3]);
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
