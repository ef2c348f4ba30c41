// kv4_attention.cuh — what the attention kernels over the paged 4-bit cache
// share: parameters, request lengths, the page cursor.
#pragma once
#include "kv4.cuh"
#include "mbarrier.cuh"

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
  int requests, tokens, group, P, page_shift;  // P = 1 << page_shift
  int max_q, max_seq, key_limit, window;  // key_limit: keys of a table row
  float scale_log2;  // softmax_scale * log2(e)
  float* partial;    // pieces of split segments
  int pad_tiles;     // decode: tiles that every request counts, 0: its own
};

// kv4_prefill.cu
int64_t prefill_workspace(int64_t d, int64_t requests, int64_t tokens, int64_t heads, int64_t group, int64_t max_q,
                          int64_t max_seq);
int prefill_launch(int dtype, int64_t d, const AttnParams& p, int64_t max_seq, cudaStream_t st);
bool prefill_timeouts(unsigned long long* count);

// First key that a row at position pos sees.  A row before position 0 sees none; with a window
// near 2^31 its pos - window would leave 32 bits.
CEK_DEVICE int first_key(const AttnParams& p, int pos) {
  return p.window > 0 ? max(max(pos, -1) + 1 - p.window, 0) : 0;
}

// What a request asks for, from its lengths.
struct Request {
  int t0, n;          // first token row, rows tokens (bounded)
  int pos0;           // position of the first token
  int tile0, live;    // tiles of TK keys that any row sees (at least one if n > 0: it writes the zeros)
  int tiles;          // the same, or the length that all requests are padded to
  int end;            // keys behind it do not exist
};
template <int TK>
CEK_DEVICE Request request_of(const AttnParams& p, int b) {
  Request r;
  r.t0 = p.query_start[b];
  const int n = max(p.query_start[b + 1] - r.t0, 0);
  const int seq = p.seq_lens[b];
  r.n = min(n, p.max_q);
  r.pos0 = max(seq, 0) - n;  // a refused request (negative): every row stands before position 0
  r.end = max(0, min(min(r.pos0 + r.n, p.max_seq), p.key_limit));
  r.tile0 = min(first_key(p, r.pos0), r.end) / TK;
  r.live = r.n > 0 ? max(1, (r.end + TK - 1) / TK - r.tile0) : 0;
  r.tiles = p.pad_tiles > 0 && r.n > 0 ? p.pad_tiles : r.live;
  return r;
}

CEK_DEVICE float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
CEK_DEVICE float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// e4m3 scales of two keys or groups as f16x2; a NaN becomes 448, so that times
// a probability of zero it is zero.
CEK_DEVICE uint32_t scales_no_nan(uint32_t pair) {
  uint32_t r;
  asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(fp8x2_to_f16x2<CEK_E4M3>(pair)), "r"(0x5F005F00u));
  return r;
}
// Whether any of 16 e4m3 bytes is NaN.
CEK_DEVICE uint32_t nan_bytes(uint4 v) {
  return (((v.x & 0x7F7F7F7Fu) + 0x01010101u) | ((v.y & 0x7F7F7F7Fu) + 0x01010101u) | ((v.z & 0x7F7F7F7Fu) + 0x01010101u) |
          ((v.w & 0x7F7F7F7Fu) + 0x01010101u)) & 0x80808080u;
}
CEK_DEVICE uint32_t lds_u32(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(a));
  return r;
}
CEK_DEVICE uint2 lds_u64(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
  return r;
}
CEK_DEVICE uint32_t lds_u16(uint32_t a) {
  uint16_t r;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(r) : "r"(a));
  return r;
}
CEK_DEVICE uint32_t lds_u8(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(r) : "r"(a));
  return r;
}

// The cursor that asks for pages: it runs ahead of the arithmetic.
// Page numbers come 32 at a time, one a lane, the next 32 asked for early.
template <int D, int TK>
struct Feeder {
  const int32_t* row;      // the request's table row
  const uint8_t* base;     // cache + head
  int tile, left, end;     // tile of the request, tiles left in the segment
  int window, ids, ids_next;

  // Tiles first, first + 1, ... of request b and kv head h; keys at or past `limit` are not read.
  CEK_DEVICE void load(const AttnParams& p, int b, int h, int first, int tiles, int limit, int lane) {
    row = p.table + (int64_t)b * p.table_stride;
    base = p.cache.data + (int64_t)h * p.cache.head_stride;
    tile = first;
    left = tiles;
    end = limit;
    window = (tile * TK) >> p.page_shift;
    ids = page_id(p, window + lane);
    ids_next = page_id(p, window + 32 + lane);
  }
  CEK_DEVICE int page_id(const AttnParams& p, int i) const {
    return ((int64_t)i << p.page_shift) < end ? min(max(__ldg(row + i), 0), p.cache.num_pages - 1) : 0;
  }
  // Page numbers of the tile at key0 are at hand after this (32 % (TK / P) == 0).
  CEK_DEVICE void look(const AttnParams& p, int key0, int lane) {
    if ((key0 >> p.page_shift) >= window + 32) {
      window += 32;
      ids = ids_next;
      ids_next = page_id(p, window + 32 + lane);
    }
  }
  // Asks for the keys (part 0) or values (1) of N tokens at key0, within the tile looked at.
  template <int N>
  CEK_DEVICE void ask_part(const AttnParams& p, uint32_t dst, uint32_t bar, int lane, int key0, int part) const {
    using L = Layout<D>;
    const int first = key0 >> p.page_shift;
    if (p.P <= N) {
      const int pages = min(N >> p.page_shift, max(0, (end - key0 + p.P - 1) >> p.page_shift));
      const int id = __shfl_sync(0xffffffffu, ids, (first - window + lane) & 31);
      const uint32_t bytes = (uint32_t)L::v_code(p.P);
      if (lane == 0) mbar::arrive_expect_tx(bar, bytes * pages);
      __syncwarp();
      if (lane < pages)
        mbar::bulk_g2s(dst + lane * bytes, base + (int64_t)id * p.cache.page_stride + part * bytes, bytes, bar);
    } else {
      const int id = __shfl_sync(0xffffffffu, ids, (first - window) & 31);
      const int off = key0 & (p.P - 1);
      const bool any = key0 < end;
      if (lane == 0) mbar::arrive_expect_tx(bar, any ? (uint32_t)L::v_code(N) : 0u);
      __syncwarp();
      if (any && lane < 2) {
        const int width = lane ? L::SCALE : L::CODE;
        const int src = part * L::v_code(p.P) + (lane ? L::k_scale(p.P) : 0) + off * width;
        mbar::bulk_g2s(dst + (lane ? L::k_scale(N) : 0), base + (int64_t)id * p.cache.page_stride + src,
                       (uint32_t)(N * width), bar);
      }
    }
  }
  // Asks for the tile, keys and values, into `dst`; the bytes complete on `bar`.
  CEK_DEVICE void ask(const AttnParams& p, uint32_t dst, uint32_t bar, int lane) {
    using L = Layout<D>;
    const int key0 = tile * TK;
    const int first = key0 >> p.page_shift;
    look(p, key0, lane);
    if (p.P <= TK) {
      const int pages = min(TK >> p.page_shift, max(0, (end - key0 + p.P - 1) >> p.page_shift));
      const int id = __shfl_sync(0xffffffffu, ids, (first - window + lane) & 31);  // TK / P divides 32
      const uint32_t bytes = (uint32_t)L::bytes(p.P);
      if (lane == 0) mbar::arrive_expect_tx(bar, bytes * pages);
      __syncwarp();
      if (lane < pages) mbar::bulk_g2s(dst + lane * bytes, base + (int64_t)id * p.cache.page_stride, bytes, bar);
    } else {
      // part of a page: its four arrays, laid out as a page of TK tokens
      const int id = __shfl_sync(0xffffffffu, ids, (first - window) & 31);
      const int off = key0 & (p.P - 1);
      const bool any = key0 < end;
      if (lane == 0) mbar::arrive_expect_tx(bar, any ? (uint32_t)L::bytes(TK) : 0u);
      __syncwarp();
      if (any && lane < 4) {
        const int width = (lane & 1) ? L::SCALE : L::CODE;
        const int src = (lane >> 1) * L::v_code(p.P) + ((lane & 1) ? L::k_scale(p.P) : 0) + off * width;
        const int to = (lane >> 1) * L::v_code(TK) + ((lane & 1) ? L::k_scale(TK) : 0);
        mbar::bulk_g2s(dst + to, base + (int64_t)id * p.cache.page_stride + src, (uint32_t)(TK * width), bar);
      }
    }
    ++tile;
    --left;
  }
};

}  // namespace kv4
}  // namespace cek
