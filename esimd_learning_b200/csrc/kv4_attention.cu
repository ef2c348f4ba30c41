// kv4_attention.cu — attention over the paged 4-bit key/value cache
// (cek_kv4_attention).
#include "kv4.cuh"

#include <algorithm>
#include <cmath>

namespace cek {
namespace kv4 {

struct AttnParams {
  const void* q;
  void* out;
  Cache cache;
  const int32_t* table;
  const int32_t* query_start;
  const int32_t* seq_lens;
  int64_t table_stride, qts, qhs, ots, ohs;
  int requests, tokens, q_heads, group, table_width, P;
  int max_q, max_seq, window;
  float scale_log2;  // softmax_scale * log2(e)
};

// One warp per (token, query head): a lane scores one key of 32, then holds
// D / 32 output channels of the weighted sum.
template <typename T, int D>
__global__ void __launch_bounds__(128)
attn_simple_kernel(const AttnParams p) {
  using L = Layout<D>;
  constexpr int E = D / 32;
  __shared__ float qs[4][D];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 4 + warp;
  const int req = blockIdx.y;
  const int t0 = p.query_start[req], t1 = min(p.query_start[req + 1], p.tokens);
  const int r = (int)(w / p.q_heads), h = (int)(w % p.q_heads);
  const int n = p.query_start[req + 1] - t0;
  if (r >= n || t0 + r >= t1 || t0 + r < 0) return;
  const int seq = p.seq_lens[req];
  const int pos = seq - n + r;
  const int end = min(min(pos + 1, p.max_seq), p.table_width * p.P);
  const int begin = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  const int kvh = h / p.group;
  const T* q = static_cast<const T*>(p.q) + (int64_t)(t0 + r) * p.qts + h * p.qhs;
  for (int i = lane; i < D; i += 32) qs[warp][i] = to_f32<T>(q[i]);
  __syncwarp();
  const float kf = p.cache.scales[kvh] * p.scale_log2, vf = p.cache.scales[p.cache.heads + kvh];
  float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int k0 = begin; k0 < end; k0 += 32) {
    const int key = k0 + lane;
    float s = -INFINITY;
    const uint8_t* block = p.cache.data;
    int off = 0;
    if (key < end) {
      const int page = min(max(p.table[req * p.table_stride + key / p.P], 0), p.cache.num_pages - 1);
      block += page * p.cache.page_stride + kvh * p.cache.head_stride;
      off = key % p.P;
      float acc = 0.f;
      for (int gidx = 0; gidx < D / 16; ++gidx) {
        const uint2 c = *reinterpret_cast<const uint2*>(block + off * L::CODE + gidx * 8);
        const float sc = e4m3_to_f32(block[L::k_scale(p.P) + off * L::SCALE + gidx]);
        float part = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const uint32_t code = ((j < 8 ? c.x : c.y) >> (4 * (j & 7))) & 15u;
          part += unpack2<__half>(e2m1x2_to_f16x2<0>(code)).x * qs[warp][gidx * 16 + j];
        }
        acc += part * sc;
      }
      s = acc * kf;
    }
    const float top = fmaxf(m, warp_max(s));
    const float base = top == -INFINITY ? 0.f : top;
    const float alpha = exp2f(m - base), pr = exp2f(s - base);
    l = l * alpha + pr;
    m = top;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= alpha;
    const int cnt = min(32, end - k0);
    for (int j = 0; j < cnt; ++j) {
      const uint8_t* bj = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, (unsigned long long)block, j));
      const int oj = __shfl_sync(0xffffffffu, off, j);
      const float pj = __shfl_sync(0xffffffffu, pr, j);
      const uint8_t* vc = bj + L::v_code(p.P) + oj * L::CODE;
      const uint8_t* vs = bj + L::v_scale(p.P) + oj * L::SCALE;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = lane * E + e;
        const uint32_t code = (vc[d >> 1] >> (4 * (d & 1))) & 15u;
        o[e] += pj * (unpack2<__half>(e2m1x2_to_f16x2<0>(code)).x * e4m3_to_f32(vs[d >> 4]));
      }
    }
  }
  l = warp_sum(l);
  T* out = static_cast<T*>(p.out) + (int64_t)(t0 + r) * p.ots + h * p.ohs;
#pragma unroll
  for (int e = 0; e < E; ++e) out[lane * E + e] = from_f32<T>(l == 0.f ? 0.f : o[e] / l * vf);
}

}  // namespace kv4
}  // namespace cek

extern "C" int64_t cek_kv4_attention_workspace_bytes(int64_t requests, int64_t tokens, int64_t q_heads,
                                                     int64_t kv_heads, int64_t head_dim, int64_t max_query_len,
                                                     int64_t max_seq_len) {
  return 0;
}

extern "C" int cek_kv4_attention(const void* query, const cek_kv4_cache* cache, const int32_t* block_table,
                                 const int32_t* query_start, const int32_t* seq_lens, void* out, void* workspace,
                                 int64_t workspace_bytes, int64_t requests, int64_t tokens, int64_t q_heads,
                                 int64_t table_width, int64_t table_stride, int64_t query_token_stride,
                                 int64_t query_head_stride, int64_t out_token_stride, int64_t out_head_stride,
                                 float softmax_scale, int64_t max_query_len, int64_t max_seq_len, int64_t window,
                                 int dtype, void* stream) {
  const int s = cek_host::kv4_check(cache);
  if (s != CEK_OK) return s;
  if (dtype != CEK_F16 && dtype != CEK_BF16) return CEK_ERR_INVALID_ARG;
  if (requests < 0 || requests > 65535 || tokens < 0 || tokens > INT32_MAX || q_heads <= 0 ||
      q_heads % cache->kv_heads || q_heads > 65535 || table_width < 0 || table_width * cache->page_size > INT32_MAX ||
      table_stride < table_width || max_query_len < 0 || max_seq_len < 0 || max_query_len > INT32_MAX ||
      max_seq_len > INT32_MAX || window < 0 || window > INT32_MAX)
    return CEK_ERR_INVALID_ARG;
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale)) return CEK_ERR_INVALID_ARG;
  if (requests == 0 || tokens == 0 || max_query_len == 0) return CEK_OK;
  if (!query || !out || !query_start || !seq_lens || (table_width > 0 && !block_table)) return CEK_ERR_INVALID_ARG;
  if (!cek_host::aligned16(query) || !cek_host::aligned16(out) || query_token_stride % 8 || query_head_stride % 8 ||
      out_token_stride % 8 || out_head_stride % 8)
    return CEK_ERR_ALIGNMENT;
  cek::kv4::AttnParams p = {};
  p.q = query;
  p.out = out;
  p.cache = cek_host::kv4_cache(cache);
  p.table = block_table;
  p.query_start = query_start;
  p.seq_lens = seq_lens;
  p.table_stride = table_stride;
  p.qts = query_token_stride;
  p.qhs = query_head_stride;
  p.ots = out_token_stride;
  p.ohs = out_head_stride;
  p.requests = (int)requests;
  p.tokens = (int)tokens;
  p.q_heads = (int)q_heads;
  p.group = (int)(q_heads / cache->kv_heads);
  p.table_width = (int)table_width;
  p.P = (int)cache->page_size;
  p.max_q = (int)std::min(max_query_len, tokens);
  p.max_seq = (int)max_seq_len;
  p.window = (int)window;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  const dim3 grid((unsigned)(((int64_t)p.max_q * q_heads + 3) / 4), (unsigned)requests), block(128);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto tag) {
    using T = decltype(tag);
    switch (cache->head_dim) {
      case 64: return cek_host::launch_pdl(cek::kv4::attn_simple_kernel<T, 64>, grid, block, 0, st, p);
      case 128: return cek_host::launch_pdl(cek::kv4::attn_simple_kernel<T, 128>, grid, block, 0, st, p);
      default: return cek_host::launch_pdl(cek::kv4::attn_simple_kernel<T, 256>, grid, block, 0, st, p);
    }
  };
  return dtype == CEK_F16 ? go(__half{}) : go(__nv_bfloat16{});
}
