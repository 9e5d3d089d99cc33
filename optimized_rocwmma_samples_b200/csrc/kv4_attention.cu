// kv4_attention.cu — attention of a few query tokens over the 4-bit cache.
//
// The queries of sequence b are its last tokens: query i of n sees positions
// below len - n + i + 1.  With keys K and values V as the cache stands for them:
//   s = scale * q . K,  p = exp(s - max s) / sum,  o = sum p V
// and, where asked, weight[head][position] += sum of p over the head's query
// heads and the queries.  A row that sees nothing gives 0.
//
// One warp per query row, positions in turn; the row's maximum and sum go to
// the workspace for the weights, which a second kernel adds up per position.
#include "kv4.cuh"

#include <algorithm>

namespace b2sq {

namespace {

struct KvAttnParams {
    Kv4Cache c;
    Kv4Seqs s;
    uint32_t heads, max_queries;
    uint64_t q_stride;
    float scale;
};

__device__ __forceinline__ float kv4_value(const uint8_t* data, const __half* sz, int64_t row, uint32_t d, uint32_t ng,
                                           uint32_t ch)
{
    const uint32_t byte = data[row * (d / 2) + ch / 2];
    const uint32_t q = (ch & 1) ? byte >> 4 : byte & 15u;
    const __half* g = sz + (row * ng + ch / kKv4Group) * 2;
    return fmaf((float)q, __half2float(g[0]), __half2float(g[1]));
}

// grid (max_queries * heads, batch), one warp a block; lane holds channels lane, lane + 32, ...
template <typename T, int D>
__global__ void __launch_bounds__(32) kv4_rows_kernel(KvAttnParams a, const T* __restrict__ q, T* __restrict__ out,
                                                      float2* __restrict__ stats)
{
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t b = blockIdx.y, i = blockIdx.x / a.heads, head = blockIdx.x % a.heads, lane = threadIdx.x;
    uint32_t start;
    const uint32_t n = kv4_new_rows(a.s, b, start);
    if (i >= n) return;
    const uint32_t kvh = head / (a.heads / a.c.kv_heads);
    const int64_t vis = (int64_t)kv4_len(a.s, b) - n + i + 1;
    const uint32_t see = (uint32_t)max((int64_t)0, min(vis, (int64_t)kv4_cap(a.c, a.s)));
    float qf[D / 32], o[D / 32];
    for (int j = 0; j < D / 32; ++j) {
        qf[j] = (float)q[(uint64_t)(start + i) * a.q_stride + (uint64_t)head * D + lane + 32 * j];
        o[j] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const int32_t* table = a.s.page_table + (uint64_t)b * a.s.max_pages;
    for (uint32_t t = 0; t < see; ++t) {
        const int64_t row = kv4_row(a.c, table, t, kvh);
        if (row < 0) continue;
        float dot = 0.f;
        for (int j = 0; j < D / 32; ++j)
            dot = fmaf(qf[j], kv4_value(a.c.k, (const __half*)a.c.k_scale, row, D, D / 64, lane + 32 * j), dot);
        for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
        const float s = dot * a.scale;
        const float mn = fmaxf(m, s), f = m == -INFINITY ? 0.f : expf(m - mn), p = s == -INFINITY ? 0.f : expf(s - mn);
        for (int j = 0; j < D / 32; ++j)
            o[j] = o[j] * f + p * kv4_value(a.c.v, (const __half*)a.c.v_scale, row, D, D / 64, lane + 32 * j);
        l = l * f + p;
        m = mn;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int j = 0; j < D / 32; ++j)
        out[((uint64_t)(start + i) * a.heads + head) * D + lane + 32 * j] = (T)(o[j] * inv);
    if (stats && lane == 0) stats[((uint64_t)b * a.max_queries + i) * a.heads + head] = make_float2(m, inv);
}

// grid (positions / 8, kv_heads, batch), a warp a position
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_weights_kernel(KvAttnParams a, const T* __restrict__ q,
                                                          const float2* __restrict__ stats)
{
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t b = blockIdx.z, kvh = blockIdx.y, t = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x & 31;
    uint32_t start;
    const uint32_t n = kv4_new_rows(a.s, b, start);
    if (t >= kv4_cap(a.c, a.s)) return;
    const int64_t row = kv4_row(a.c, a.s.page_table + (uint64_t)b * a.s.max_pages, t, kvh);
    const uint32_t group = a.heads / a.c.kv_heads;
    float sum = 0.f;
    bool any = false;
    for (uint32_t i = 0; i < min(n, a.max_queries); ++i) {
        if ((int64_t)t >= (int64_t)kv4_len(a.s, b) - n + i + 1 || row < 0) continue;
        any = true;
        for (uint32_t g = 0; g < group; ++g) {
            const uint32_t head = kvh * group + g;
            float dot = 0.f;
            for (int j = 0; j < D / 32; ++j)
                dot = fmaf((float)q[(uint64_t)(start + i) * a.q_stride + (uint64_t)head * D + lane + 32 * j],
                           kv4_value(a.c.k, (const __half*)a.c.k_scale, row, D, D / 64, lane + 32 * j), dot);
            for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
            const float2 st = stats[((uint64_t)b * a.max_queries + i) * a.heads + head];
            sum += expf(dot * a.scale - st.x) * st.y;
        }
    }
    if (lane == 0 && any) a.c.weight[row] += sum;
}

template <typename T, int D>
cudaError_t run(const Kv4Attention& a, void* workspace, cudaStream_t st)
{
    const KvAttnParams p{a.cache, a.seqs, a.heads, a.max_queries, a.q_stride, a.scale};
    float2* stats = a.accumulate ? static_cast<float2*>(workspace) : nullptr;
    cudaError_t e = launch_pdl(kv4_rows_kernel<T, D>, dim3(a.max_queries * a.heads, a.seqs.batch), dim3(32), 0, st, p,
                               static_cast<const T*>(a.q), static_cast<T*>(a.out), stats);
    if (e != cudaSuccess || !a.accumulate) return e;
    const uint32_t cap = a.seqs.max_pages * a.cache.page_size;
    return launch_pdl(kv4_weights_kernel<T, D>, dim3((cap + 7) / 8, a.cache.kv_heads, a.seqs.batch), dim3(256), 0, st,
                      p, static_cast<const T*>(a.q), static_cast<const float2*>(stats));
}

}  // namespace

size_t kv4_attention_workspace(uint32_t batch, uint32_t heads, uint32_t, uint32_t, uint32_t max_queries, uint32_t,
                               bool accumulate, uint32_t)
{
    return accumulate ? (size_t)batch * heads * max_queries * sizeof(float2) : 0;
}

cudaError_t launch_kv4_attention(const Kv4Attention& a, void* workspace, uint32_t, cudaStream_t st)
{
    switch (a.cache.head_dim) {
        case 64: return a.bf16 ? run<__nv_bfloat16, 64>(a, workspace, st) : run<__half, 64>(a, workspace, st);
        case 128: return a.bf16 ? run<__nv_bfloat16, 128>(a, workspace, st) : run<__half, 128>(a, workspace, st);
        default: return a.bf16 ? run<__nv_bfloat16, 256>(a, workspace, st) : run<__half, 256>(a, workspace, st);
    }
}

}  // namespace b2sq
