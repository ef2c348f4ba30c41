// kv4_cache.cu — the paged 4-bit key/value cache around its attention:
//   * page plan of a step from request lengths   (cek_kv_plan)
//   * quantise new tokens into the cache         (cek_kv4_append)
//   * read tokens back in 16 bits                (cek_kv4_gather)
#include "kv4.cuh"

#include <algorithm>

namespace cek {
namespace kv4 {

// ---- append ------------------------------------------------------------------
// One thread per 16-channel group of one token and head, keys and values in one
// grid.  The D/16 threads of a head lie side by side in a warp: their code
// bytes are one contiguous store, their scale bytes are gathered into one.
template <typename T, bool VEC>
CEK_DEVICE void load_group(const T* p, float (&x)[16]) {
  if constexpr (VEC) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 v = ldg_nc(p + 8 * h);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(w[i]);
        x[8 * h + 2 * i] = f.x;
        x[8 * h + 2 * i + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = to_f32<T>(p[i]);
  }
}

template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(256)
append_kernel(const T* __restrict__ key, const T* __restrict__ value, const int64_t* __restrict__ slots, Cache c,
              int P, int64_t groups, int64_t kts, int64_t khs, int64_t vts, int64_t vhs) {
  using L = Layout<D>;
  constexpr int GP = D / 16;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const bool live = id < groups;
  const int64_t u = live ? id : groups - 1;
  const int grp = (int)(u % GP);
  const int64_t head_row = u / GP;                 // (token, k or v, head)
  const int h = (int)(head_row % c.heads);
  const int64_t r = head_row / c.heads;
  const int kv = (int)(r & 1);
  const int64_t t = r >> 1;
  const int64_t slot = slots[t];
  const bool store = live && slot >= 0 && slot < (int64_t)c.num_pages * P;
  const T* src = kv ? value + t * vts + h * vhs : key + t * kts + h * khs;
  float x[16];
  load_group<T, VEC>(src + grp * 16, x);
  float a = 0.f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    a = fmaxf(a, fabsf(x[i]));  // fmaxf drops a NaN: remembered beside it
    nan |= x[i] != x[i];
  }
  if (nan) a = __int_as_float(0x7fffffff);
  const float g = c.scales[kv * c.heads + h];
  const uint32_t s8 = __nv_cvt_float_to_fp8(__fdiv_rn(a, __fmul_rn(6.f, g)), __NV_SATFINITE, __NV_E4M3);
  const float unit = __fmul_rn(e4m3_to_f32(s8), g);
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 y = make_float2(unit == 0.f ? 0.f : __fdiv_rn(x[2 * i], unit),
                                 unit == 0.f ? 0.f : __fdiv_rn(x[2 * i + 1], unit));
    w[i >> 2] |= (uint32_t)__nv_cvt_float2_to_fp4x2(y, __NV_E2M1, cudaRoundNearest) << (8 * (i & 3));
  }
  // scale bytes of the head: 4 groups a word, collected in the first of each four lanes
  uint32_t sw = s8 << (8 * (grp & 3));
  sw |= __shfl_xor_sync(0xffffffffu, sw, 1);
  sw |= __shfl_xor_sync(0xffffffffu, sw, 2);
  if (!store) return;
  const int64_t page = slot / P;
  const int off = (int)(slot % P);
  uint8_t* block = c.data + page * c.page_stride + (int64_t)h * c.head_stride;
  *reinterpret_cast<uint2*>(block + (kv ? L::v_code(P) : 0) + off * L::CODE + grp * 8) = make_uint2(w[0], w[1]);
  if ((grp & 3) == 0)
    *reinterpret_cast<uint32_t*>(block + (kv ? L::v_scale(P) : L::k_scale(P)) + off * L::SCALE + grp) = sw;
}

// ---- gather ------------------------------------------------------------------
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(256)
gather_kernel(Cache c, const int64_t* __restrict__ slots, T* __restrict__ key, T* __restrict__ value, int P,
              int64_t groups, int64_t kts, int64_t khs, int64_t vts, int64_t vhs) {
  using L = Layout<D>;
  constexpr int GP = D / 16;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (id >= groups) return;
  const int grp = (int)(id % GP);
  const int64_t head_row = id / GP;
  const int h = (int)(head_row % c.heads);
  const int64_t r = head_row / c.heads;
  const int kv = (int)(r & 1);
  const int64_t t = r >> 1;
  const int64_t slot = slots[t];
  uint2 w = make_uint2(0u, 0u);
  float s = 0.f;
  if (slot >= 0 && slot < (int64_t)c.num_pages * P) {
    const uint8_t* block = c.data + (slot / P) * c.page_stride + (int64_t)h * c.head_stride;
    const int off = (int)(slot % P);
    w = *reinterpret_cast<const uint2*>(block + (kv ? L::v_code(P) : 0) + off * L::CODE + grp * 8);
    s = e4m3_to_f32(block[(kv ? L::v_scale(P) : L::k_scale(P)) + off * L::SCALE + grp]);
  }
  const float g = c.scales[kv * c.heads + h];
  const uint32_t pr[8] = {e2m1x2_to_f16x2<0>(w.x), e2m1x2_to_f16x2<1>(w.x), e2m1x2_to_f16x2<2>(w.x),
                          e2m1x2_to_f16x2<3>(w.x), e2m1x2_to_f16x2<0>(w.y), e2m1x2_to_f16x2<1>(w.y),
                          e2m1x2_to_f16x2<2>(w.y), e2m1x2_to_f16x2<3>(w.y)};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = unpack2<__half>(pr[i]);
    o[i] = pack2<T>(__fmul_rn(f.x * s, g), __fmul_rn(f.y * s, g));
  }
  T* dst = (kv ? value + t * vts + h * vhs : key + t * kts + h * khs) + grp * 16;
  if constexpr (VEC) {
    reinterpret_cast<uint4*>(dst)[0] = make_uint4(o[0], o[1], o[2], o[3]);
    reinterpret_cast<uint4*>(dst)[1] = make_uint4(o[4], o[5], o[6], o[7]);
  } else {
    const T* e = reinterpret_cast<const T*>(o);
#pragma unroll
    for (int i = 0; i < 16; ++i) dst[i] = e[i];
  }
}

// ---- page plan -----------------------------------------------------------------
// One cluster of up to 8 CTAs.  Every CTA scans the request lengths by itself
// (a block scan of two sums; requests <= 4096), the cluster's barrier then
// separates the last read of context_lens and free_count from the first write
// of seq_lens and free_count_out (they may be the same arrays), and the CTAs
// share the table entries and the tokens.
constexpr int kPlanThreads = 1024;
constexpr int kPlanTokensPerCta = 2048;

CEK_DEVICE int pages_of(int tokens, int P) { return (int)(((int64_t)tokens + P - 1) / P); }

__global__ void __launch_bounds__(kPlanThreads)
plan_kernel(const int32_t* __restrict__ query_lens, const int32_t* context_lens, int32_t* block_table,
            const int32_t* __restrict__ free_pages, const int32_t* free_count, int32_t* __restrict__ query_start,
            int32_t* seq_lens, int32_t* free_count_out, int64_t* __restrict__ positions, int64_t* __restrict__ slots,
            int B, int W, int64_t table_stride, int pool, int64_t tokens, int P) {
  extern __shared__ int32_t sm[];
  int32_t* start = sm;               // [B + 1] first token of each request
  int32_t* taken = sm + B + 1;       // [B] pages taken before request i; negative: refused
  int32_t* ctx = sm + 2 * B + 1;     // [B]
  __shared__ int2 warp_sums[32];
  __shared__ int carry_q, carry_n, granted_pages;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t rank, ctas;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  if (tid == 0) carry_q = carry_n = granted_pages = 0;
  const int avail = min(max(*free_count, 0), pool);
  __syncthreads();
  for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int i = b0 + tid;
    int q = 0, c = -1, need = 0;
    bool fits = false;
    if (i < B) {
      q = max(query_lens[i], 0);
      c = context_lens[i];
      if (c >= 0) {
        const int have = pages_of(c, P), all = (int)(((int64_t)c + q + P - 1) / P);
        fits = all <= W;
        need = fits ? all - have : 0;
      }
    }
    int sq = q, sn = need;  // inclusive scans
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, sq, o), b = __shfl_up_sync(0xffffffffu, sn, o);
      if (lane >= o) { sq += a; sn += b; }
    }
    if (lane == 31) warp_sums[warp] = make_int2(sq, sn);
    __syncthreads();
    if (warp == 0) {
      int2 v = warp_sums[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, v.x, o), b = __shfl_up_sync(0xffffffffu, v.y, o);
        if (lane >= o) { v.x += a; v.y += b; }
      }
      warp_sums[lane] = v;
    }
    __syncthreads();
    if (warp > 0) { sq += warp_sums[warp - 1].x; sn += warp_sums[warp - 1].y; }
    sq += carry_q;
    sn += carry_n;
    if (i < B) {
      const bool granted = fits && (need == 0 || sn <= avail);
      start[i] = sq - q;
      taken[i] = granted ? sn - need : -1;
      ctx[i] = c;
      if (granted && need > 0) atomicMax(&granted_pages, sn);  // a maximum: the order does not matter
    }
    __syncthreads();
    if (tid == kPlanThreads - 1) { carry_q = sq; carry_n = sn; }
    __syncthreads();
  }
  if (tid == 0) start[B] = carry_q;
  // all of the cluster has read context_lens and free_count
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  __syncthreads();
  const int stride = (int)ctas * kPlanThreads, gid = (int)rank * kPlanThreads + tid;
  if (gid == 0) free_count_out[0] = avail - granted_pages;
  for (int i = gid; i <= B; i += stride) {
    query_start[i] = start[i];
    if (i < B) {
      const int c = ctx[i];
      seq_lens[i] = taken[i] >= 0 ? c + (start[i + 1] - start[i]) : (c < 0 ? c : ~c);
    }
  }
  // new table entries: a warp per request
  for (int i = gid >> 5; i < B; i += stride >> 5) {
    if (taken[i] < 0) continue;
    const int have = pages_of(ctx[i], P), need = pages_of(ctx[i] + (start[i + 1] - start[i]), P) - have;
    for (int j = lane; j < need; j += 32)
      block_table[(int64_t)i * table_stride + have + j] = free_pages[avail - 1 - (taken[i] + j)];
  }
  const int total = start[B];
  for (int64_t t = gid; t < tokens; t += stride) {
    int64_t position = 0, slot = -1;
    if (t < total) {
      int lo = 0, hi = B - 1;  // the last request whose first token is not behind t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start[mid] <= (int)t) lo = mid; else hi = mid - 1;
      }
      const int c = ctx[lo], pos = (c < 0 ? ~c : c) + (int)t - start[lo];
      position = pos;
      if (taken[lo] >= 0) {
        const int have = pages_of(c, P), pg = pos / P;
        const int page = pg < have ? block_table[(int64_t)lo * table_stride + pg]
                                   : free_pages[avail - 1 - (taken[lo] + pg - have)];
        slot = (int64_t)page * P + pos % P;
      }
    }
    positions[t] = position;
    slots[t] = slot;
  }
}

}  // namespace kv4
}  // namespace cek

extern "C" int64_t cek_kv4_page_bytes(int64_t page_size, int64_t head_dim) {
  if (!cek_host::kv4_page_size(page_size) || !cek_host::kv4_head_dim(head_dim)) return 0;
  return page_size * (head_dim + head_dim / 8);
}

extern "C" int cek_kv_plan(const int32_t* query_lens, const int32_t* context_lens, int32_t* block_table,
                           const int32_t* free_pages, const int32_t* free_count, int32_t* query_start,
                           int32_t* seq_lens, int32_t* free_count_out, int64_t* positions, int64_t* slot_mapping,
                           int64_t requests, int64_t table_width, int64_t table_stride, int64_t pool_size,
                           int64_t tokens, int64_t page_size, void* stream) {
  if (requests < 0 || requests > CEK_KV_PLAN_MAX_REQUESTS || table_width < 0 || table_width > INT32_MAX ||
      table_stride < table_width || pool_size < 0 || pool_size > INT32_MAX || tokens < 0 || tokens > INT32_MAX ||
      page_size < 1 || page_size > INT32_MAX / 2)
    return CEK_ERR_INVALID_ARG;
  if (!free_count || !query_start || !free_count_out) return CEK_ERR_INVALID_ARG;
  if (requests > 0 && (!query_lens || !context_lens || !seq_lens || (table_width > 0 && !block_table)))
    return CEK_ERR_INVALID_ARG;
  if ((tokens > 0 && (!positions || !slot_mapping)) || (pool_size > 0 && !free_pages)) return CEK_ERR_INVALID_ARG;
  const int smem = (int)(sizeof(int32_t) * (3 * requests + 1));
  static cek_host::DeviceSlots slots_attr;
  if (smem > 48 * 1024 - 1024 &&
      !cek_host::ensure_smem_attr(slots_attr, cek::kv4::plan_kernel, (int)sizeof(int32_t) * (3 * CEK_KV_PLAN_MAX_REQUESTS + 1)))
    return CEK_ERR_LAUNCH;
  // CTAs by the tokens to write; a portable cluster has 8 at most
  const int ctas = (int)std::min<int64_t>(8, std::max<int64_t>(1, (tokens + cek::kv4::kPlanTokensPerCta - 1) /
                                                                      cek::kv4::kPlanTokensPerCta));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(cek::kv4::kPlanThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = cek_host::pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, cek::kv4::plan_kernel, query_lens, context_lens, block_table, free_pages, free_count,
                            query_start, seq_lens, free_count_out, positions, slot_mapping, (int)requests,
                            (int)table_width, table_stride, (int)pool_size, tokens, (int)page_size) == cudaSuccess
             ? CEK_OK
             : CEK_ERR_LAUNCH;
}

namespace {
template <typename T>
bool vec_ok(const T* p, int64_t ts, int64_t hs) { return cek_host::aligned16(p) && ts % 8 == 0 && hs % 8 == 0; }

// 0: launch; otherwise the status to return (*done) for bad or empty arguments
int token_args(const void* key, const void* value, const int64_t* slots, const cek_kv4_cache* cache, int64_t tokens,
               int dtype, bool* done) {
  *done = true;
  const int s = cek_host::kv4_check(cache);
  if (s != CEK_OK) return s;
  if (tokens < 0 || (dtype != CEK_F16 && dtype != CEK_BF16)) return CEK_ERR_INVALID_ARG;
  if (tokens == 0) return CEK_OK;
  if (!key || !value || !slots) return CEK_ERR_INVALID_ARG;
  if (tokens * 2 * cache->kv_heads * (cache->head_dim / 16) > (int64_t)INT32_MAX * 256) return CEK_ERR_INVALID_ARG;
  *done = false;
  return CEK_OK;
}
}  // namespace

#define CEK_KV4_DISPATCH(KERNEL, A0, A1, A2, A3)                                                                     \
  do {                                                                                                               \
    const int64_t groups = tokens * 2 * cache->kv_heads * (cache->head_dim / 16);                                    \
    const dim3 grid((unsigned)((groups + 255) / 256)), block(256);                                                   \
    cudaStream_t st = static_cast<cudaStream_t>(stream);                                                             \
    const bool vec = vec_ok(key, key_token_stride, key_head_stride) &&                                               \
                     vec_ok(value, value_token_stride, value_head_stride);                                           \
    const int P = (int)cache->page_size;                                                                             \
    auto go = [&](auto tag, auto dim, auto v) {                                                                      \
      using T = decltype(tag);                                                                                       \
      return cek_host::launch_pdl(cek::kv4::KERNEL<T, decltype(dim)::value, decltype(v)::value>, grid, block, 0, st, \
                                  A0, A1, A2, A3, P, groups, key_token_stride, key_head_stride, value_token_stride,  \
                                  value_head_stride);                                                                \
    };                                                                                                               \
    auto by_vec = [&](auto tag, auto dim) { return vec ? go(tag, dim, std::true_type{}) : go(tag, dim, std::false_type{}); }; \
    auto by_dim = [&](auto tag) {                                                                                    \
      switch (cache->head_dim) {                                                                                     \
        case 64: return by_vec(tag, std::integral_constant<int, 64>{});                                              \
        case 128: return by_vec(tag, std::integral_constant<int, 128>{});                                            \
        default: return by_vec(tag, std::integral_constant<int, 256>{});                                             \
      }                                                                                                              \
    };                                                                                                               \
    return dtype == CEK_F16 ? by_dim(__half{}) : by_dim(__nv_bfloat16{});                                            \
  } while (0)

extern "C" int cek_kv4_append(const void* key, const void* value, const int64_t* slot_mapping,
                              const cek_kv4_cache* cache, int64_t tokens, int64_t key_token_stride,
                              int64_t key_head_stride, int64_t value_token_stride, int64_t value_head_stride,
                              int dtype, void* stream) {
  bool done;
  const int s = token_args(key, value, slot_mapping, cache, tokens, dtype, &done);
  if (done) return s;
  const cek::kv4::Cache c = cek_host::kv4_cache(cache);
  CEK_KV4_DISPATCH(append_kernel, static_cast<const T*>(key), static_cast<const T*>(value), slot_mapping, c);
}

extern "C" int cek_kv4_gather(const cek_kv4_cache* cache, const int64_t* slots, void* key, void* value, int64_t tokens,
                              int64_t key_token_stride, int64_t key_head_stride, int64_t value_token_stride,
                              int64_t value_head_stride, int dtype, void* stream) {
  bool done;
  const int s = token_args(key, value, slots, cache, tokens, dtype, &done);
  if (done) return s;
  const cek::kv4::Cache c = cek_host::kv4_cache(cache);
  CEK_KV4_DISPATCH(gather_kernel, c, slots, static_cast<T*>(key), static_cast<T*>(value));
}
