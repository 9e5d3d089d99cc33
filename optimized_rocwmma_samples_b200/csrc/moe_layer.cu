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
// Four plain kernels: quantise x, one warp per (route, gate and up row),
// quantise h, one warp per (token, output).
#include "common.cuh"
#include "kernels.h"
#include "sq_math.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2sq {

namespace {

constexpr uint32_t kThreads = 256;

__device__ __forceinline__ float block_max(float v)
{
    __shared__ float part[kThreads / 32];
    for (int off = 16; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    v = part[0];
    for (uint32_t i = 1; i < kThreads / 32; ++i) v = fmaxf(v, part[i]);
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) moe_quant_x(MoeLayer m, int8_t* xq, float* rs)
{
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t r = blockIdx.x;
    const int32_t e = m.topk_ids[r];
    if ((uint32_t)e >= m.experts) return;
    const T* x = static_cast<const T*>(m.x) + (r / m.topk) * m.x_stride;
    const float* s = m.smooth1 + (uint64_t)e * m.hidden;
    float mx = 0.f;
    for (uint32_t i = threadIdx.x; i < m.hidden; i += kThreads) mx = fmaxf(mx, fabsf(__fmul_rn((float)x[i], s[i])));
    const float sc = row_scale_of(block_max(mx), m.qmax), inv = inv_scale_of(sc);
    for (uint32_t i = threadIdx.x; i < m.hidden; i += kThreads)
        xq[(uint64_t)r * m.hidden + i] = quant1(__fmul_rn((float)x[i], s[i]), inv, m.qmax);
    if (threadIdx.x == 0) rs[r] = sc;
}

__device__ __forceinline__ int warp_dot(const int8_t* a, const int8_t* b, uint32_t k, uint32_t lane)
{
    int acc = 0;
    const int4* av = reinterpret_cast<const int4*>(a);
    const int4* bv = reinterpret_cast<const int4*>(b);
    for (uint32_t i = lane; i < k / 16; i += 32) {
        const int4 x = av[i], y = bv[i];
        acc = __dp4a(x.x, y.x, acc);
        acc = __dp4a(x.y, y.y, acc);
        acc = __dp4a(x.z, y.z, acc);
        acc = __dp4a(x.w, y.w, acc);
    }
    for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
    return acc;
}

__global__ void __launch_bounds__(kThreads) moe_gate_up(MoeLayer m, const int8_t* xq, const float* rs, float* h)
{
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t r = blockIdx.y, j = blockIdx.x * (kThreads / 32) + threadIdx.x / 32, lane = threadIdx.x & 31;
    const int32_t e = m.topk_ids[r];
    if ((uint32_t)e >= m.experts || j >= m.inter) return;
    const int8_t* w = m.w13 + (uint64_t)e * 2 * m.inter * m.hidden;
    const int8_t* x = xq + (uint64_t)r * m.hidden;
    const float* s = m.s13 + (uint64_t)e * 2 * m.inter;
    const float g = (float)warp_dot(w + (uint64_t)j * m.hidden, x, m.hidden, lane) * (rs[r] * s[j]);
    const float u = (float)warp_dot(w + (uint64_t)(m.inter + j) * m.hidden, x, m.hidden, lane) * (rs[r] * s[m.inter + j]);
    if (lane == 0) h[(uint64_t)r * m.inter + j] = g / (1.f + expf(-g)) * u * m.smooth2[(uint64_t)e * m.inter + j];
}

__global__ void __launch_bounds__(kThreads) moe_quant_h(MoeLayer m, const float* h, int8_t* hq, float* rs)
{
    griddep_wait();
    griddep_launch_dependents();
    const uint64_t r = blockIdx.x;
    if ((uint32_t)m.topk_ids[r] >= m.experts) return;
    float mx = 0.f;
    for (uint32_t i = threadIdx.x; i < m.inter; i += kThreads) mx = fmaxf(mx, fabsf(h[r * m.inter + i]));
    const float sc = row_scale_of(block_max(mx), m.qmax), inv = inv_scale_of(sc);
    for (uint32_t i = threadIdx.x; i < m.inter; i += kThreads) hq[r * m.inter + i] = quant1(h[r * m.inter + i], inv, m.qmax);
    if (threadIdx.x == 0) rs[r] = sc;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) moe_down(MoeLayer m, const int8_t* hq, const float* rs)
{
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t t = blockIdx.y, i = blockIdx.x * (kThreads / 32) + threadIdx.x / 32, lane = threadIdx.x & 31;
    if (i >= m.hidden) return;
    float sum = 0.f;
    for (uint32_t k = 0; k < m.topk; ++k) {
        const uint64_t r = (uint64_t)t * m.topk + k;
        const int32_t e = m.topk_ids[r];
        if ((uint32_t)e >= m.experts) continue;
        const uint64_t row = (uint64_t)e * m.hidden + i;
        const int acc = warp_dot(m.w2 + row * m.inter, hq + r * m.inter, m.inter, lane);
        sum = fmaf(m.topk_w[r], (float)acc * (rs[r] * m.s2[row]), sum);
    }
    if (lane == 0) static_cast<T*>(m.out)[(uint64_t)t * m.hidden + i] = (T)sum;
}

struct Ws {
    float *h, *rs1, *rs2;
    int8_t *xq, *hq;
    size_t bytes;
};
Ws carve(const MoeLayer& m, void* base)
{
    const size_t r = (size_t)m.tokens * m.topk;
    uint8_t* p = static_cast<uint8_t*>(base);
    size_t at = 0;
    auto take = [&](size_t n) {
        uint8_t* q = p + at;
        at += (n + 255) / 256 * 256;
        return q;
    };
    Ws w;
    w.h = reinterpret_cast<float*>(take(r * m.inter * 4));
    w.xq = reinterpret_cast<int8_t*>(take(r * m.hidden));
    w.hq = reinterpret_cast<int8_t*>(take(r * m.inter));
    w.rs1 = reinterpret_cast<float*>(take(r * 4));
    w.rs2 = reinterpret_cast<float*>(take(r * 4));
    w.bytes = at;
    return w;
}

template <typename T>
cudaError_t run(const MoeLayer& m, void* workspace, cudaStream_t st)
{
    const Ws w = carve(m, workspace);
    const uint32_t r = m.tokens * m.topk;
    constexpr uint32_t kWarps = kThreads / 32;
    cudaError_t e = launch_pdl(moe_quant_x<T>, dim3(r), dim3(kThreads), 0, st, m, w.xq, w.rs1);
    if (e == cudaSuccess)
        e = launch_pdl(moe_gate_up, dim3((m.inter + kWarps - 1) / kWarps, r), dim3(kThreads), 0, st, m, (const int8_t*)w.xq,
                       (const float*)w.rs1, w.h);
    if (e == cudaSuccess) e = launch_pdl(moe_quant_h, dim3(r), dim3(kThreads), 0, st, m, (const float*)w.h, w.hq, w.rs2);
    if (e == cudaSuccess)
        e = launch_pdl(moe_down<T>, dim3((m.hidden + kWarps - 1) / kWarps, m.tokens), dim3(kThreads), 0, st, m,
                       (const int8_t*)w.hq, (const float*)w.rs2);
    return e;
}

}  // namespace

size_t moe_layer_workspace(uint32_t tokens, uint32_t hidden, uint32_t inter, uint32_t experts, uint32_t topk, uint32_t)
{
    MoeLayer m{};
    m.tokens = tokens, m.hidden = hidden, m.inter = inter, m.experts = experts, m.topk = topk;
    return carve(m, nullptr).bytes;
}

cudaError_t launch_moe_layer(const MoeLayer& m, void* workspace, uint32_t, cudaStream_t st)
{
    return m.bf16 ? run<__nv_bfloat16>(m, workspace, st) : run<__half>(m, workspace, st);
}

}  // namespace b2sq
