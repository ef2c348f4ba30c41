// kv4_cache.cu — the paged 4-bit key/value cache around its attention:
//   * page plan of a step from request lengths   (cek_kv_plan)
//   * quantise new tokens into the cache         (cek_kv4_append)
//   * read tokens back in 16 bits                (cek_kv4_gather)
#include "kv4.cuh"

#include <algorithm>
#include <type_traits>

namespace cek {
namespace kv4 {

// ---- append and gather -------------------------------------------------------
// Both move 16-bit values on one side and 4.5 bits a value on the other: HBM is
// their bound, and the instructions around 16 bytes are what competes with it.
// A gather thread takes 8 channels, 16 bytes of the 16-bit side, of both the key
// and the value of a unit (token, head): D/8 neighbouring lanes have a unit,
// every access of a warp is contiguous, and a unit's place is worked out once.
// An append thread takes a whole group of 16, so that the scale is worked out
// once.  Long calls give a thread U = 2 units, their loads in flight together;
// short ones one, for more threads (kManyAppend, kManyGather).
// 32 769 tokens of 8 heads of 128 read back: 32.2 us, 5.4 TB/s (82 % of a copy; with
// integer divisions by page and head count it was 41).  8191 tokens written: 10.2 us,
// 4.2 TB/s; 65 % of the issue slots are taken, most by the quotients (20 us with a
// division a channel).
template <typename T, bool VEC>
CEK_DEVICE uint4 load8(const T* p) {
  if constexpr (VEC) return ldg_nc(p);
  const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = e[2 * i] | ((uint32_t)e[2 * i + 1] << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T, bool VEC>
CEK_DEVICE void store8(T* p, uint4 v) {
  if constexpr (VEC) {
    *reinterpret_cast<uint4*>(p) = v;
  } else {
    uint16_t* e = reinterpret_cast<uint16_t*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[2 * i] = (uint16_t)w[i];
      e[2 * i + 1] = (uint16_t)(w[i] >> 16);
    }
  }
}

// Division of n < 2^31 by a number that the launch fixes, as a multiplication:
// n / d = (mulhi(n, m) + n) >> s with s = ceil(log2 d), m = floor(2^32 (2^s - d) / d) + 1.
struct Divisor {
  uint32_t d, m, s;
  explicit Divisor(uint32_t d_) : d(d_), s(0) {
    while ((1ull << s) < d) ++s;
    m = (uint32_t)((((1ull << s) - d) << 32) / d) + 1;
  }
};
CEK_DEVICE uint32_t divide(uint32_t n, const Divisor& d) { return (__umulhi(n, d.m) + n) >> d.s; }
// Unit number -> token, head.
CEK_DEVICE int2 token_head(uint32_t u, const Divisor& n) {
  const uint32_t t = divide(u, n);
  return make_int2((int)t, (int)(u - t * n.d));
}

// Codes and scale byte of a group of 16 channels.
template <typename T>
CEK_DEVICE uint2 quantize16(const uint4 (&v)[2], float g, uint32_t& s8) {
  const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
  // largest magnitude: 16-bit patterns without their sign order as their values, a NaN above infinity
  uint32_t mx = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) mx = __vmaxu2(mx, w[j] & 0x7FFF7FFFu);
  const float a = unpack2<T>(max(mx & 0xFFFFu, mx >> 16)).x;
  s8 = __nv_cvt_float_to_fp8(__fdiv_rn(a, __fmul_rn(6.f, g)), __NV_SATFINITE, __NV_E4M3);
  const float unit = __fmul_rn(e4m3_to_f32(s8), g);
  uint32_t code[2] = {0, 0};
  if (unit > 0x1p-60f && unit < 0x1p60f && a < 0x1p100f) {
    // x / unit correctly rounded without a division per channel, as in
    // quant_fp8_per_token_kernel (Markstein: the correctly rounded reciprocal and
    // two corrections), two channels an instruction.  On -x, so that the
    // remainder q unit - x of a zero is +0 and the quotient keeps its sign.
    const float y = __frcp_rn(unit);
    const uint64_t n2 = f32x2(-y, -y), u2 = f32x2(unit, unit);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 x = unpack2<T>(w[j] ^ 0x80008000u);
      const uint64_t x2 = f32x2(x.x, x.y);
      uint64_t q = mul_f32x2(x2, n2);
      q = fma_f32x2(fma_f32x2(q, u2, x2), n2, q);
      q = fma_f32x2(fma_f32x2(q, u2, x2), n2, q);
      float2 r;
      unpack_f32x2(q, r.x, r.y);
      code[j >> 2] |= (uint32_t)__nv_cvt_float2_to_fp4x2(r, __NV_E2M1, cudaRoundNearest) << (8 * (j & 3));
    }
  } else {
    // a unit far from 1 (or zero, or NaN)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 x = unpack2<T>(w[j]);
      const float2 r = make_float2(unit == 0.f ? 0.f : __fdiv_rn(x.x, unit), unit == 0.f ? 0.f : __fdiv_rn(x.y, unit));
      code[j >> 2] |= (uint32_t)__nv_cvt_float2_to_fp4x2(r, __NV_E2M1, cudaRoundNearest) << (8 * (j & 3));
    }
  }
  return make_uint2(code[0], code[1]);
}

template <typename T, int D, bool VEC, int U>
__global__ void __launch_bounds__(256)
append_kernel(const T* __restrict__ key, const T* __restrict__ value, const int64_t* __restrict__ slots, Cache c,
              int shift, uint32_t units, const Divisor heads, int64_t kts, int64_t khs, int64_t vts, int64_t vhs) {
  using L = Layout<D>;
  constexpr int LANES = D / 16, PER = 256 / LANES;
  const int P = 1 << shift;
  pdl_launch_dependents();
  pdl_wait();
  const int ln = threadIdx.x % LANES;  // its group of 16 channels
  const uint32_t u0 = blockIdx.x * (PER * U) + threadIdx.x / LANES;
  uint4 x[U][2][2];  // [unit][k, v][halves]
  int64_t slot[U];
  int h[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const uint32_t u = u0 + i * PER;
    const int2 n = token_head(min(u, units - 1), heads);
    h[i] = n.y;
    slot[i] = u < units ? slots[n.x] : -1;
    const T* k = key + (int64_t)n.x * kts + n.y * khs + ln * 16;
    const T* v = value + (int64_t)n.x * vts + n.y * vhs + ln * 16;
    x[i][0][0] = load8<T, VEC>(k);
    x[i][0][1] = load8<T, VEC>(k + 8);
    x[i][1][0] = load8<T, VEC>(v);
    x[i][1][1] = load8<T, VEC>(v + 8);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const bool store = slot[i] >= 0 && slot[i] < (int64_t)c.num_pages << shift;
    uint8_t* block = c.data + (store ? (slot[i] >> shift) * c.page_stride + (int64_t)h[i] * c.head_stride : 0);
    const int off = (int)slot[i] & (P - 1);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint32_t s8;
      const uint2 code = quantize16<T>(x[i][kv], c.scales[kv * c.heads + h[i]], s8);
      // the scales of four groups as one word
      s8 <<= 8 * (ln & 3);
      s8 |= __shfl_xor_sync(0xffffffffu, s8, 1);
      s8 |= __shfl_xor_sync(0xffffffffu, s8, 2);
      if (!store) continue;
      uint8_t* part = block + (kv ? L::v_code(P) : 0);
      *reinterpret_cast<uint2*>(part + off * L::CODE + ln * 8) = code;
      if ((ln & 3) == 0) *reinterpret_cast<uint32_t*>(part + P * L::CODE + off * L::SCALE + ln) = s8;
    }
  }
}

// 8 values from their codes and scale byte: code * scale is exact in fp16.
template <typename T>
CEK_DEVICE uint4 values8(uint32_t code, uint32_t s8, float g) {
  const uint32_t s = __byte_perm(fp8x2_to_f16x2<CEK_E4M3>(s8), 0, 0x1010);
  const uint32_t p[4] = {hmul2(e2m1x2_to_f16x2<0>(code), s), hmul2(e2m1x2_to_f16x2<1>(code), s),
                         hmul2(e2m1x2_to_f16x2<2>(code), s), hmul2(e2m1x2_to_f16x2<3>(code), s)};
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = unpack2<__half>(p[j]);
    o[j] = pack2<T>(__fmul_rn(f.x, g), __fmul_rn(f.y, g));
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <typename T, int D, bool VEC, int U>
__global__ void __launch_bounds__(256)
gather_kernel(Cache c, const int64_t* __restrict__ slots, T* __restrict__ key, T* __restrict__ value, int shift,
              uint32_t units, const Divisor heads, int64_t kts, int64_t khs, int64_t vts, int64_t vhs) {
  using L = Layout<D>;
  constexpr int LANES = D / 8, PER = 256 / LANES;
  const int P = 1 << shift;
  pdl_launch_dependents();
  pdl_wait();
  const int ln = threadIdx.x % LANES;
  const uint32_t u0 = blockIdx.x * (PER * U) + threadIdx.x / LANES;
  int64_t slot[U];
  int2 n[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    n[i] = token_head(min(u0 + i * PER, units - 1), heads);
    slot[i] = slots[n[i].x];
  }
  uint32_t kc[U], vc[U], ks[U], vs[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    kc[i] = vc[i] = ks[i] = vs[i] = 0;
    if (slot[i] < 0 || slot[i] >= (int64_t)c.num_pages << shift) continue;
    const uint8_t* block = c.data + (slot[i] >> shift) * c.page_stride + (int64_t)n[i].y * c.head_stride;
    const int off = (int)slot[i] & (P - 1), code = off * L::CODE + ln * 4, sca = P * L::CODE + off * L::SCALE + (ln >> 1);
    kc[i] = __ldg(reinterpret_cast<const uint32_t*>(block + code));
    ks[i] = __ldg(block + sca);
    vc[i] = __ldg(reinterpret_cast<const uint32_t*>(block + L::v_code(P) + code));
    vs[i] = __ldg(block + L::v_code(P) + sca);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (u0 + i * PER >= units) continue;
    store8<T, VEC>(key + (int64_t)n[i].x * kts + n[i].y * khs + ln * 8, values8<T>(kc[i], ks[i], c.scales[n[i].y]));
    store8<T, VEC>(value + (int64_t)n[i].x * vts + n[i].y * vhs + ln * 8,
                   values8<T>(vc[i], vs[i], c.scales[c.heads + n[i].y]));
  }
}

// ---- page plan -----------------------------------------------------------------
// One cluster of up to 16 CTAs, one small CTA for a step of few tokens.  Every
// CTA scans the request lengths by itself (a block scan of two sums; requests <=
// 4096), the cluster's barrier then
// separates the last read of context_lens and free_count from the first write
// of seq_lens and free_count_out (they may be the same arrays), and the CTAs
// share the table entries and the tokens.  1000 requests with 64 000 tokens: 8.8 us
// (13.5 on 8 CTAs with divisions); 64 requests of one token: 4.3 us.
constexpr int kPlanThreads = 1024;
constexpr int kPlanTokensPerCta = 2048;
constexpr int kPlanBatch = 4;

CEK_DEVICE int pages_of(int tokens, const Divisor& P) {
  const uint32_t full = divide((uint32_t)tokens, P);
  return (int)(full + (full * P.d != (uint32_t)tokens));
}

// For N ascending searches at once: the last i in [0, n) with a[i] <= x, their
// shared-memory loads in flight together.  a[0] <= x.
template <int N>
CEK_DEVICE void last_not_above(const int32_t* a, int n, const int (&x)[N], int (&at)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) at[k] = 0;
  for (int step = 1 << (31 - __clz(n)); step > 0; step >>= 1) {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (at[k] + step < n && a[at[k] + step] <= x[k]) at[k] += step;
  }
}

__global__ void __launch_bounds__(kPlanThreads)
plan_kernel(const int32_t* __restrict__ query_lens, const int32_t* context_lens, int32_t* block_table,
            const int32_t* __restrict__ free_pages, const int32_t* free_count, int32_t* __restrict__ query_start,
            int32_t* seq_lens, int32_t* free_count_out, int64_t* __restrict__ positions, int64_t* __restrict__ slots,
            int B, int W, int64_t table_stride, int pool, int64_t tokens, const Divisor P) {
  extern __shared__ int32_t sm[];
  int32_t* start = sm;               // [B + 1] first token of each request
  int32_t* asked = sm + B + 1;       // [B + 1] pages asked for before each request
  int32_t* ctx = sm + 2 * B + 2;     // [B] tokens that its pages hold; their complement (negative) if refused
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
  const int64_t row_tokens = min((int64_t)W * P.d, (int64_t)INT32_MAX);
  const int threads = blockDim.x, warps = threads >> 5;
  for (int b0 = 0; b0 < B; b0 += threads) {
    const int i = b0 + tid;
    int q = 0, c = -1, need = 0;
    bool fits = false;
    if (i < B) {
      q = max(query_lens[i], 0);
      c = context_lens[i];
      if (c >= 0) {
        // c + q may leave 32 bits; where it fits the row it does not
        fits = (int64_t)c + q <= row_tokens;
        need = fits ? pages_of(c + q, P) - pages_of(c, P) : 0;
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
      int2 v = lane < warps ? warp_sums[lane] : make_int2(0, 0);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, v.x, o), b = __shfl_up_sync(0xffffffffu, v.y, o);
        if (lane >= o) { v.x += a; v.y += b; }
      }
      if (lane < warps) warp_sums[lane] = v;
    }
    __syncthreads();
    if (warp > 0) { sq += warp_sums[warp - 1].x; sn += warp_sums[warp - 1].y; }
    sq += carry_q;
    sn += carry_n;
    if (i < B) {
      const bool granted = fits && (need == 0 || sn <= avail);
      start[i] = sq - q;
      asked[i] = sn - need;
      ctx[i] = granted ? c : c < 0 ? c : ~c;
      if (granted && need > 0) atomicMax(&granted_pages, sn);  // a maximum: the order does not matter
    }
    __syncthreads();
    if (tid == threads - 1) { carry_q = sq; carry_n = sn; }
    __syncthreads();
  }
  if (tid == 0) {
    start[B] = carry_q;
    asked[B] = carry_n;
  }
  // all of the cluster has read context_lens and free_count
  if (ctas > 1) asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  __syncthreads();
  const int stride = (int)ctas * threads, gid = (int)rank * threads + tid;
  if (gid == 0) free_count_out[0] = avail - granted_pages;
  for (int i = gid; i <= B; i += stride) {
    query_start[i] = start[i];
    if (i < B) seq_lens[i] = ctx[i] >= 0 ? ctx[i] + (start[i + 1] - start[i]) : ctx[i];
  }
  // new table entries: entry e of the line of all pages asked for
  const int entries = B > 0 ? min(asked[B], avail) : 0;
  for (int e = gid; e < entries; e += stride) {
    const int x[1] = {e};
    int at[1];
    last_not_above<1>(asked, B, x, at);
    const int i = at[0], c = ctx[i];
    if (c >= 0) block_table[(int64_t)i * table_stride + pages_of(c, P) + e - asked[i]] = free_pages[avail - 1 - e];
  }
  // tokens, kPlanBatch a thread at once
  const int total = start[B];
  constexpr int N = kPlanBatch;
  for (int64_t t0 = gid; t0 < tokens; t0 += (int64_t)stride * N) {
    int x[N], at[N];
    int64_t slot[N], position[N];
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = (int)min(t0 + (int64_t)k * stride, (int64_t)INT32_MAX);
    if (B > 0) last_not_above<N>(start, B, x, at);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      slot[k] = -1;
      position[k] = 0;
      if (x[k] >= total || x[k] >= tokens) continue;
      const int i = at[k], c = ctx[i];
      position[k] = (int64_t)(c < 0 ? ~c : c) + (x[k] - start[i]);
      if (c >= 0) {
        const int pos = (int)position[k];
        const int have = pages_of(c, P), pg = (int)divide((uint32_t)pos, P);
        const int page = pg < have ? block_table[(int64_t)i * table_stride + pg] : free_pages[avail - 1 - (asked[i] + pg - have)];
        slot[k] = (int64_t)page * P.d + (pos - pg * (int)P.d);
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (x[k] < tokens) {
        positions[x[k]] = position[k];
        slots[x[k]] = slot[k];
      }
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
  const int smem = (int)(sizeof(int32_t) * (3 * requests + 2));
  static cek_host::DeviceSlots slots_attr;
  if (smem > 48 * 1024 - 1024 &&
      !cek_host::ensure_smem_attr(slots_attr, cek::kv4::plan_kernel, (int)sizeof(int32_t) * (3 * CEK_KV_PLAN_MAX_REQUESTS + 2)))
    return CEK_ERR_LAUNCH;
  // CTAs by the tokens to write; above 8 a cluster is not portable, but this is one GPU's code
  const int ctas = (int)std::min<int64_t>(16, std::max<int64_t>(1, (tokens + cek::kv4::kPlanTokensPerCta - 1) /
                                                                       cek::kv4::kPlanTokensPerCta));
  const int threads = requests <= 256 && tokens <= 1024 ? 256 : cek::kv4::kPlanThreads;
  if (ctas > 8) {
    static cek_host::DeviceSlots wide;
    int dev = 0;
    cudaGetDevice(&dev);
    std::atomic<int>* done = wide.at(dev);
    if (!done || !done->load(std::memory_order_relaxed)) {
      if (cudaFuncSetAttribute(cek::kv4::plan_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return CEK_ERR_LAUNCH;
      if (done) done->store(1, std::memory_order_relaxed);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3((unsigned)threads);
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
                            (int)table_width, table_stride, (int)pool_size, tokens, cek::kv4::Divisor((uint32_t)page_size)) == cudaSuccess
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
  if (tokens > INT32_MAX) return CEK_ERR_INVALID_ARG;
  *done = false;
  return CEK_OK;
}
}  // namespace

// Blocks an SM (of one unit a thread) above which a thread takes two.  Device time, one and
// two units, 8 heads of 128 (64 and 256 channels turn within a step of the same place):
//   blocks an SM      4           8           16          32          64          128
//   append, us    5.1 / 4.6   6.9 / 7.6  11.4 / 12.4  20.9 / 21.5  39.7 / 39.8  76.9 / 76.0
//   gather, us    2.7 / 2.8   3.7 / 3.6   6.8 / 6.5   12.1 / 11.2  22.3 / 19.6  42.4 / 36.5
// An append thread has work enough of its own between its loads; a gather thread has not.
// (Append's half microsecond at 4 blocks, gone at 8, is not worth a second turn.)
constexpr int64_t kManyAppend = 64, kManyGather = 8;

// Launches KERNEL on [tokens], in parts whose unit numbers stay below 2^31.
#define CEK_KV4_DISPATCH(KERNEL, CHANNELS, MANY, A0, A1, A2, A3)                                                     \
  do {                                                                                                               \
    const int64_t per = 256 / (cache->head_dim / CHANNELS), row = cache->kv_heads;                                      \
    cudaStream_t st = static_cast<cudaStream_t>(stream);                                                             \
    const bool vec = vec_ok(key, key_token_stride, key_head_stride) &&                                               \
                     vec_ok(value, value_token_stride, value_head_stride);                                           \
    const cek::kv4::Divisor heads((uint32_t)cache->kv_heads);                                                          \
    int shift = 0;                                                                                                   \
    while ((1 << shift) < cache->page_size) ++shift;                                                                 \
    const int64_t part = ((1ll << 31) - 4096) / row;                                                                 \
    int rc = CEK_OK;                                                                                                 \
    for (int64_t t0 = 0; t0 < tokens && rc == CEK_OK; t0 += part) {                                                  \
      const uint32_t units = (uint32_t)(std::min(part, tokens - t0) * row);                                          \
      const bool many = units > per * MANY * cek_host::sm_count();                                                   \
      const dim3 grid((unsigned)((units + per * (many ? 2 : 1) - 1) / (per * (many ? 2 : 1)))), block(256);          \
      auto go = [&](auto tag, auto dim, auto v) {                                                                    \
        using T = decltype(tag);                                                                                     \
        constexpr int D = decltype(dim)::value;                                                                      \
        constexpr bool V = decltype(v)::value;                                                                       \
        auto run = [&](auto kern) {                                                                                  \
          return cek_host::launch_pdl(kern, grid, block, 0, st, A0, A1, A2, A3, shift, units, heads,                 \
                                      key_token_stride, key_head_stride, value_token_stride, value_head_stride);     \
        };                                                                                                           \
        return many ? run(cek::kv4::KERNEL<T, D, V, 2>) : run(cek::kv4::KERNEL<T, D, V, 1>);                         \
      };                                                                                                             \
      auto by_vec = [&](auto tag, auto dim) {                                                                        \
        return vec ? go(tag, dim, std::true_type{}) : go(tag, dim, std::false_type{});                               \
      };                                                                                                             \
      auto by_dim = [&](auto tag) {                                                                                  \
        switch (cache->head_dim) {                                                                                   \
          case 64: return by_vec(tag, std::integral_constant<int, 64>{});                                            \
          case 128: return by_vec(tag, std::integral_constant<int, 128>{});                                          \
          default: return by_vec(tag, std::integral_constant<int, 256>{});                                           \
        }                                                                                                            \
      };                                                                                                             \
      rc = dtype == CEK_F16 ? by_dim(__half{}) : by_dim(__nv_bfloat16{});                                            \
    }                                                                                                                \
    return rc;                                                                                                       \
  } while (0)

extern "C" int cek_kv4_append(const void* key, const void* value, const int64_t* slot_mapping,
                              const cek_kv4_cache* cache, int64_t tokens, int64_t key_token_stride,
                              int64_t key_head_stride, int64_t value_token_stride, int64_t value_head_stride,
                              int dtype, void* stream) {
  bool done;
  const int s = token_args(key, value, slot_mapping, cache, tokens, dtype, &done);
  if (done) return s;
  const cek::kv4::Cache c = cek_host::kv4_cache(cache);
  CEK_KV4_DISPATCH(append_kernel, 16, kManyAppend, static_cast<const T*>(key) + t0 * key_token_stride,
                   static_cast<const T*>(value) + t0 * value_token_stride, slot_mapping + t0, c);
}

extern "C" int cek_kv4_gather(const cek_kv4_cache* cache, const int64_t* slots, void* key, void* value, int64_t tokens,
                              int64_t key_token_stride, int64_t key_head_stride, int64_t value_token_stride,
                              int64_t value_head_stride, int dtype, void* stream) {
  bool done;
  const int s = token_args(key, value, slots, cache, tokens, dtype, &done);
  if (done) return s;
  const cek::kv4::Cache c = cek_host::kv4_cache(cache);
  CEK_KV4_DISPATCH(gather_kernel, 8, kManyGather, c, slots + t0, static_cast<T*>(key) + t0 * key_token_stride,
                   static_cast<T*>(value) + t0 * value_token_stride);
}
