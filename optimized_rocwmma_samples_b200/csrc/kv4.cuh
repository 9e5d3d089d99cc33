// kv4.cuh — the paged key/value cache held in 4 bits, shared by the kernels
// that write it (kv4_append.cu), read it (kv4_attention.cu) and thin it out
// (kv4_evict.cu).
//
// A token's keys (and values) in one head are D channels in groups of 64.  A
// group holds 64 nibbles q, a step s and a base z (both fp16): value = q s + z.
//   k, v             [pages][kv_heads][page_size][D / 2]  channel 2i in the low nibble of byte i
//   k_scale, v_scale [pages][kv_heads][page_size][D / 64] pairs (s, z)
//   weight           [pages][kv_heads][page_size]         accumulated attention weight (nullable)
// Position p of sequence b is slot p % page_size of page page_table[b][p / page_size].
#pragma once

#include "common.cuh"
#include "sq_math.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2sq {

constexpr uint32_t kKv4Group = 64;

// Row (page, head, slot) of the cache; -1 where the table names no page of it.
__device__ __forceinline__ int64_t kv4_row(const Kv4Cache& c, const int32_t* __restrict__ table_row, uint32_t pos,
                                           uint32_t head)
{
    const uint32_t at = c.page_shift >= 0 ? pos >> c.page_shift : pos / c.page_size;
    const int32_t page = __ldg(table_row + at);
    if ((uint32_t)page >= c.pages) return -1;
    return ((int64_t)page * c.kv_heads + head) * c.page_size + (pos - at * c.page_size);
}

// Length of sequence b (negative lengths count as 0); only its first kv4_cap tokens have a place in the table.
__device__ __forceinline__ uint32_t kv4_len(const Kv4Seqs& s, uint32_t b)
{
    return (uint32_t)max(__ldg(s.seq_lens + b), 0);
}
__device__ __forceinline__ uint32_t kv4_cap(const Kv4Cache& c, const Kv4Seqs& s) { return s.max_pages * c.page_size; }

// Rows [start, start + count) of the packed tokens that belong to sequence b.
// Offsets that leave [0, tokens] or run backwards count as an empty sequence.
__device__ __forceinline__ uint32_t kv4_new_rows(const Kv4Seqs& s, uint32_t b, uint32_t& start)
{
    const int32_t t0 = __ldg(s.token_start + b), t1 = __ldg(s.token_start + b + 1);
    start = (uint32_t)t0;
    return (t0 < 0 || t1 < t0 || (uint32_t)t1 > s.tokens) ? 0u : (uint32_t)(t1 - t0);
}

template <typename T>
__device__ __forceinline__ float2 pair_to_f2(uint32_t w);
template <>
__device__ __forceinline__ float2 pair_to_f2<__half>(uint32_t w)
{
    float2 f;
    h2_to_f2(w, f.x, f.y);
    return f;
}
template <>
__device__ __forceinline__ float2 pair_to_f2<__nv_bfloat16>(uint32_t w)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t f2_to_pair(float a, float b);
template <>
__device__ __forceinline__ uint32_t f2_to_pair<__half>(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t f2_to_pair<__nv_bfloat16>(float a, float b)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace b2sq
