// kv4.cuh — the paged 4-bit key/value cache: block layout and decoding.
//
// cache [pages, kv heads, page bytes], P tokens of D channels a page.  One
// (page, head) block, a multiple of 16 bytes, holds
//   K codes [P, D/2] | K scales [P, D/16] | V codes [P, D/2] | V scales [P, D/16]
// so everything that attention reads of a page is one contiguous range.  A
// code is an e2m1 number (channel 2i in the low four bits of byte i); 16
// channels of a token share one e4m3 scale; kv_scales [2, heads] fp32 spans
// the range that e4m3 does not.
//
// code * scale has at most 6 significant bits and lies in [2^-10, 2688], so
// it is exact in fp16: the matrix instructions get the stored values without
// a rounding, and kv_scales is applied in fp32 afterwards.
#pragma once
#include "common.cuh"

#include <cuda_fp4.h>
#include <cuda_fp8.h>

namespace cek {
namespace kv4 {

struct Cache {
  uint8_t* data;
  const float* scales;  // [2, heads]
  int64_t page_stride, head_stride;  // bytes
  int num_pages, heads;
};

template <int D>
struct Layout {
  static constexpr int CODE = D / 2, SCALE = D / 16;  // bytes per token
  __host__ __device__ static constexpr int k_scale(int P) { return P * CODE; }
  __host__ __device__ static constexpr int v_code(int P) { return P * (CODE + SCALE); }
  __host__ __device__ static constexpr int v_scale(int P) { return P * (2 * CODE + SCALE); }
  __host__ __device__ static constexpr int bytes(int P) { return P * 2 * (CODE + SCALE); }
};

// Two codes (one byte; byte `b` of w) -> f16x2, low half = the low four bits.
template <int B>
CEK_DEVICE uint32_t e2m1x2_to_f16x2(uint32_t w) {
  uint32_t r;
  if constexpr (B == 0)
    asm("{ .reg .b8 a, b, c, d; mov.b32 {a, b, c, d}, %1; cvt.rn.f16x2.e2m1x2 %0, a; }" : "=r"(r) : "r"(w));
  else if constexpr (B == 1)
    asm("{ .reg .b8 a, b, c, d; mov.b32 {a, b, c, d}, %1; cvt.rn.f16x2.e2m1x2 %0, b; }" : "=r"(r) : "r"(w));
  else if constexpr (B == 2)
    asm("{ .reg .b8 a, b, c, d; mov.b32 {a, b, c, d}, %1; cvt.rn.f16x2.e2m1x2 %0, c; }" : "=r"(r) : "r"(w));
  else
    asm("{ .reg .b8 a, b, c, d; mov.b32 {a, b, c, d}, %1; cvt.rn.f16x2.e2m1x2 %0, d; }" : "=r"(r) : "r"(w));
  return r;
}
CEK_DEVICE uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Two fp32 numbers in one register pair: one instruction for both.
CEK_DEVICE uint64_t f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
CEK_DEVICE void unpack_f32x2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
CEK_DEVICE uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
CEK_DEVICE uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
CEK_DEVICE uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// One e4m3 byte -> fp32 (exact; NaN codes -> NaN).
CEK_DEVICE float e4m3_to_f32(uint32_t b) {
  const uint32_t h = fp8x2_to_f16x2<CEK_E4M3>(b & 0xFFu);
  return unpack2<__half>(h).x;
}

}  // namespace kv4
}  // namespace cek

// Host side: the argument checks that the entry points share.
namespace cek_host {
inline bool kv4_head_dim(int64_t d) { return d == 64 || d == 128 || d == 256; }
inline bool kv4_page_size(int64_t p) { return p == 16 || p == 32 || p == 64 || p == 128; }
// CEK_OK, or why `c` cannot be used.
inline int kv4_check(const cek_kv4_cache* c) {
  if (!c || !kv4_head_dim(c->head_dim) || !kv4_page_size(c->page_size)) return CEK_ERR_INVALID_ARG;
  if (c->num_pages <= 0 || c->num_pages > INT32_MAX || c->kv_heads <= 0 || c->kv_heads > 65535) return CEK_ERR_INVALID_ARG;
  if (!c->data || !c->scales) return CEK_ERR_INVALID_ARG;
  const int64_t block = cek_kv4_page_bytes(c->page_size, c->head_dim);
  if (c->head_stride < block && c->kv_heads > 1) return CEK_ERR_INVALID_ARG;
  if (c->page_stride < block && c->num_pages > 1) return CEK_ERR_INVALID_ARG;
  if (!aligned16(c->data) || c->page_stride % 16 || c->head_stride % 16) return CEK_ERR_ALIGNMENT;
  return CEK_OK;
}
inline cek::kv4::Cache kv4_cache(const cek_kv4_cache* c) {
  return {static_cast<uint8_t*>(c->data), c->scales, c->page_stride, c->head_stride, (int)c->num_pages, (int)c->kv_heads};
}
}  // namespace cek_host
