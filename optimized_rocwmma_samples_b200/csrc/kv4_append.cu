// kv4_append.cu — writes new keys and values into the 4-bit paged cache.
//
// Per group of 64 channels (v saturated to fp16's finite range):
//   z = fp16(min v), s = fp16((max v - min v) / 15)
//   q = clamp(rint((v - z) / s), 0, 15), ties to even; s = 0 gives q = 0
// A NaN makes its group's s and z NaN, so it is not lost in the cache.
//
// Bound by HBM (2 bytes a channel in, 0.56 out, 2 more where the cached
// values are asked for): eight lanes hold a group, one 16-byte load and one
// 4-byte store of nibbles each, the extrema by three shuffles.  The quotient
// is a product with 1 / s corrected by its exact remainder, since inputs of
// 8 or 11 significant bits meet the border between two steps often.
#include "kv4.cuh"

namespace b2sq {

namespace {

constexpr uint32_t kAppendThreads = 256;
constexpr float kHalfMax = 65504.f;

template <typename T>
__global__ void __launch_bounds__(kAppendThreads)
    kv4_append_kernel(Kv4Cache c, Kv4Seqs s, const T* __restrict__ k, const T* __restrict__ v, uint64_t k_stride,
                      uint64_t v_stride, T* __restrict__ k_out, T* __restrict__ v_out)
{
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t ng = c.head_dim / kKv4Group;
    const uint32_t per_token = c.kv_heads * ng;  // groups
    const uint64_t total = (uint64_t)s.tokens * per_token;
    const uint64_t gi = ((uint64_t)blockIdx.x * kAppendThreads + threadIdx.x) / 8;
    if (gi >= total) return;  // the eight lanes of a group leave together
    const bool is_v = blockIdx.y != 0;
    const uint32_t lane8 = threadIdx.x & 7;
    const uint32_t mask = 0xffu << (threadIdx.x & 24);
    const uint32_t token = (uint32_t)(gi / per_token), in_token = (uint32_t)(gi % per_token);

    // the sequence that holds this token: the last one starting at or before it
    uint32_t lo = 0, hi = s.batch;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (__ldg(s.token_start + mid + 1) <= (int32_t)token)
            lo = mid + 1;
        else
            hi = mid;
    }
    if (lo == s.batch) return;
    uint32_t start;
    const uint32_t count = kv4_new_rows(s, lo, start);
    if (token < start || token - start >= count) return;
    // the new tokens are the sequence's last ones; what falls outside the table is not written
    const int64_t p = (int64_t)kv4_len(s, lo) - count + (token - start);
    if (p < 0 || p >= (int64_t)kv4_cap(c, s)) return;
    const uint32_t head = in_token / ng, g = in_token % ng;
    const int64_t row = kv4_row(c, s.page_table + (uint64_t)lo * s.max_pages, (uint32_t)p, head);
    if (row < 0) return;

    const uint64_t ch = (uint64_t)in_token * kKv4Group + lane8 * 8;
    const uint4 raw = *reinterpret_cast<const uint4*>((is_v ? v + token * v_stride : k + token * k_stride) + ch);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float f[8];
    float mn = kHalfMax, mx = -kHalfMax;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = pair_to_f2<T>(w[i]);
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        nan |= f[i] != f[i];
        f[i] = fminf(fmaxf(f[i], -kHalfMax), kHalfMax);
        mn = fminf(mn, f[i]);
        mx = fmaxf(mx, f[i]);
    }
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) {
        mn = fminf(mn, __shfl_xor_sync(mask, mn, off));
        mx = fmaxf(mx, __shfl_xor_sync(mask, mx, off));
    }
    nan = __any_sync(mask, nan);
    const __half sh = __float2half_rn((mx - mn) / 15.f), zh = __float2half_rn(mn);
    const float step = __half2float(sh), base = __half2float(zh);
    const float inv = step > 0.f ? 1.f / step : 0.f;
    uint32_t packed = 0;
    float back[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = f[i] - base;
        float q = rintf(t * inv);
        const float r2 = 2.f * fmaf(-q, step, t);  // twice the exact remainder
        const bool odd = ((int)q & 1) != 0;
        if (r2 > step || (r2 == step && odd)) q += 1.f;
        if (r2 < -step || (r2 == -step && odd)) q -= 1.f;
        q = step > 0.f ? fminf(fmaxf(q, 0.f), 15.f) : 0.f;
        packed |= (uint32_t)q << (4 * i);
        back[i] = nan ? __int_as_float(0x7fffffff) : fmaf(q, step, base);
    }
    uint8_t* data = (is_v ? c.v : c.k) + row * (c.head_dim / 2);
    reinterpret_cast<uint32_t*>(data)[g * 8 + lane8] = packed;
    if (lane8 == 0) {
        const uint32_t sz = nan ? 0x7fff7fffu : (uint32_t)__half_as_ushort(sh) | ((uint32_t)__half_as_ushort(zh) << 16);
        reinterpret_cast<uint32_t*>(is_v ? c.v_scale : c.k_scale)[row * ng + g] = sz;
        if (!is_v && g == 0 && c.weight) c.weight[row] = 0.f;
    }
    T* out = is_v ? v_out : k_out;
    if (out) {
        uint4 o;
        o.x = f2_to_pair<T>(back[0], back[1]);
        o.y = f2_to_pair<T>(back[2], back[3]);
        o.z = f2_to_pair<T>(back[4], back[5]);
        o.w = f2_to_pair<T>(back[6], back[7]);
        *reinterpret_cast<uint4*>(out + (uint64_t)token * c.kv_heads * c.head_dim + ch) = o;
    }
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4Cache& c, const Kv4Seqs& s, const void* k, const void* v, bool bf16,
                              uint64_t k_stride, uint64_t v_stride, void* k_out, void* v_out, cudaStream_t st)
{
    const uint64_t groups = (uint64_t)s.tokens * c.kv_heads * (c.head_dim / kKv4Group);
    const dim3 grid((uint32_t)((groups * 8 + kAppendThreads - 1) / kAppendThreads), 2);
    if (bf16)
        return launch_pdl(kv4_append_kernel<__nv_bfloat16>, grid, dim3(kAppendThreads), 0, st, c, s,
                          static_cast<const __nv_bfloat16*>(k), static_cast<const __nv_bfloat16*>(v), k_stride,
                          v_stride, static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out));
    return launch_pdl(kv4_append_kernel<__half>, grid, dim3(kAppendThreads), 0, st, c, s,
                      static_cast<const __half*>(k), static_cast<const __half*>(v), k_stride, v_stride,
                      static_cast<__half*>(k_out), static_cast<__half*>(v_out));
}

}  // namespace b2sq
