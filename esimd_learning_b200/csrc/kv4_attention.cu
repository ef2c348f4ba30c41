// kv4_attention.cu — attention over the paged 4-bit key/value cache
// (cek_kv4_attention).
#include "kv4_attention.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace cek {
namespace kv4 {

// ---- decode ------------------------------------------------------------------
// Few rows a request (single tokens, drafted tokens): the cache is read once
// and HBM is the bound; what has to keep up is turning 4-bit codes into matrix
// operands.
//
//  * A warp is a worker with a ring of its own in shared memory: it asks for
//    the pages of its next tiles (TK keys; one bulk copy a page, since a
//    (page, head) block is contiguous) and computes on the oldest one.  No
//    barrier between warps until the end.
//  * The tiles of all (request, kv head, row block) segments form one line, cut
//    into equal ranges: ragged lengths cost no idle time.  A segment inside one
//    range is written out by its worker; the pieces of the others (running
//    maximum, sum, unnormalised output) become one in shared memory where a CTA
//    has a part of one segment only, and go to the workspace, where
//    attn_join_kernel adds them in the order of the keys.
//  * S^T = K Q^T and O^T = V^T P^T: keys (channels) are the 16 rows of
//    mma.sync m16n8k16, up to 8 NT query rows its columns, so 8 heads of a
//    group waste nothing.  Lane (g, t) of a warp reads the codes of key g's
//    channels [t D/4, (t+1) D/4) in 16 bytes; the order of channels within the
//    sum is free as long as the query's fragments have the same.
//  * codes become f16x2 by cvt (two codes), times the group's scale: exact
//    (kv4.cuh).  A value fragment pairs two keys of one channel: the words of two
//    keys are interleaved nibble by nibble before the conversion, two
//    operations for four pairs.
//  * Key row r of a 16-key block is key (r & 8) + ((r & 7) >> 1) + 4 (r & 1):
//    then the value lanes of one access read four neighbouring keys.
//  * The probabilities of a tile, rounded to fp16, turn into the second
//    product's operand by movmatrix.  They are held as 2^kShift p, so that fp16
//    keeps full precision down to p = 2^-28.  fp16 because a matrix operand has 16
//    bits and this type the most of them; the sum of the probabilities is fp32.
//  * bf16 queries are scaled by a power of two a row, exactly, into fp16's
//    range: one multiply path for both types (what falls out below is 2^-38 of
//    the row's largest channel).
//
// Bound: latency.  A tile of 64 keys of 128 channels is ~1180 instructions of a
// scheduler (256 conversions, 256 scalings and 64 matrix instructions among them)
// and takes it ~2300 cycles, where HBM would deliver it in 1580.  No pipe is full
// (issue slots 50 %, ALU 44 %, tensor 19 %, DRAM 44 %): three warps a scheduler, what
// the registers allow, mostly wait for their own last instruction.  More warps on
// tiles of 32 keys or two accumulators for S did not help, fewer integer
// instructions did.  131 071 keys of 64/8 heads of 128, one token: 47 us,
// 3.2 TB/s with start and join (4.6 TB/s in between); 64 ragged requests to 8192
// keys: 88 us, 3.8 TB/s; 17 keys: 6 us.
constexpr float kShift = 14.f;
constexpr int kDecodeWarps = 4;
constexpr int kDecodeThreads = 32 * kDecodeWarps;
constexpr int kMaxRequests = 2048;  // per launch: their prefix sums sit in shared memory
constexpr uint32_t kWaitPolls = 1u << 22;

__device__ unsigned long long g_timeouts;

// Keys of a tile, CTAs of an SM (what the registers allow) and stages of a
// warp's ring (what then fits into 228 KB).
template <int D, int NT>
struct DecodeCfg {
  static constexpr int TK = D == 256 ? 32 : 64;
  static constexpr int STAGE = Layout<D>::bytes(TK);
  static constexpr int PER_SM = D == 64 ? (NT == 1 ? 4 : 3) : D == 128 ? (NT == 1 ? 3 : 2) : 2;
  static constexpr int STAGES = D == 64 ? (NT == 1 ? 3 : 4) : D == 128 ? (NT == 1 ? 2 : 3) : 3;
  static constexpr int RING = kDecodeWarps * STAGES * STAGE;
};

struct Segment {
  int b, h, rb;
  Request r;
  int first, tiles;  // its tiles are [first, first + tiles) of the line
};

// prefix[b] = tiles of the requests before b, all heads and row blocks
template <int TK, int ROWS>
CEK_DEVICE Segment segment_at(const AttnParams& p, const int32_t* prefix, int tile) {
  int lo = 0, hi = p.requests - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= tile) lo = mid; else hi = mid - 1;
  }
  Segment s;
  s.b = lo;
  s.r = request_of<TK>(p, lo);
  s.tiles = s.r.tiles;
  const int rbs = (s.r.n * p.group + ROWS - 1) / ROWS;
  const int idx = (tile - prefix[lo]) / s.tiles;
  s.h = idx / rbs;  // the row blocks of a head side by side: they read the same pages
  s.rb = idx % rbs;
  s.first = prefix[lo] + idx * s.tiles;
  return s;
}

// Exclusive sums of the requests' tiles into prefix[0 .. requests]; the whole block calls it.
template <int TK, int ROWS>
CEK_DEVICE void scan_requests(const AttnParams& p, int32_t* prefix, int32_t* warp_sum) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  int carry = 0;
  for (int b0 = 0; b0 < p.requests; b0 += blockDim.x) {
    const int b = b0 + tid;
    int v = 0;
    if (b < p.requests) {
      const Request r = request_of<TK>(p, b);
      v = r.tiles * p.cache.heads * ((r.n * p.group + ROWS - 1) / ROWS);
    }
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += a;
    }
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    int before = carry, all = 0;
    for (int w = 0; w < warps; ++w) {
      if (w < warp) before += warp_sum[w];
      all += warp_sum[w];
    }
    if (b < p.requests) prefix[b] = before + s - v;
    carry += all;
    __syncthreads();
  }
  if (tid == 0) prefix[p.requests] = carry;
  __syncthreads();
}

// Ranges of the line: CTA c has tiles [c S, (c + 1) S), its warps four near-equal
// parts.  S is at least a tile a warp, so that a CTA's pieces of a long segment
// become one in shared memory.  Short segments (one or two tiles a warp, padded to
// one length) are never cut: a CTA has one of them, or each of its warps whole ones.
struct Ranges {
  int total, share;
  CEK_DEVICE Ranges(int total_, int share_) : total(total_), share(share_) {}
  CEK_DEVICE static int share_of(int total, int ctas, int pad) {
    if (pad == 0) return max(kDecodeWarps, (total + ctas - 1) / ctas);
    int segments = (total / pad + ctas - 1) / ctas;
    if (segments > 1) segments = (segments + kDecodeWarps - 1) / kDecodeWarps * kDecodeWarps;
    return max(1, segments) * pad;
  }
  CEK_DEVICE int at(int cta, int warp) const { return min(total, cta * share + share * warp / kDecodeWarps); }
  CEK_DEVICE int cta_of(int tile) const { return tile / share; }
  // The whole CTA is inside the segment: its warps' pieces become one.
  CEK_DEVICE bool merged(int cta, int first, int end) const {
    const int a = at(cta, 0), b = at(cta, kDecodeWarps);
    return a + 1 < b && first <= a && b <= end;
  }
  // Where the piece of a segment is kept: a warp has a slot for its first
  // segment and one for its last; a merged CTA uses its first warp's.
  CEK_DEVICE int slot(int cta, int warp, int first, bool is_merged) const {
    return is_merged ? 2 * kDecodeWarps * cta : 2 * (kDecodeWarps * cta + warp) + (first > at(cta, warp) ? 1 : 0);
  }
};

// What the join has to know of a segment that starts in a warp's part and goes
// beyond it (one a warp at most); rows = 0: none.  In front of the pieces.
struct JoinItem {
  int first, end, total, share;  // the segment's tiles, all tiles, a CTA's
  int t0, h, row0, rows;         // first token, kv head, the row block's first row, the kv head's rows
};

CEK_DEVICE uint32_t movmatrix_t(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
CEK_DEVICE void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kDecodeThreads, (DecodeCfg<D, NT>::PER_SM))
attn_decode_kernel(const AttnParams p) {
  using C = DecodeCfg<D, NT>;
  using L = Layout<D>;
  constexpr int TK = C::TK, ROWS = 8 * NT, MT = TK / 16;
  constexpr int WORDS = D / 32;       // 4-byte code words of a lane's share of a key
  constexpr int STEPS = D / 16;       // k16 steps of the first product
  constexpr int VW = D / 64;          // code words of a lane's channels of a value
  constexpr int MI = 4 * VW;          // 16-channel row tiles of the second product
  constexpr int VG = D == 256 ? 2 : 1;  // scale groups among a lane's value channels
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kDecodeWarps][C::STAGES];
  __shared__ int32_t warp_sums[kDecodeWarps];
  int32_t* prefix = reinterpret_cast<int32_t*>(smem + C::RING);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  pdl_launch_dependents();
  if (lane == 0) {
    for (int s = 0; s < C::STAGES; ++s) mbar::init(mbar::saddr(&bars[warp][s]), 1);
    mbar::fence_init();
  }
  pdl_wait();
  scan_requests<TK, ROWS>(p, prefix, warp_sums);
  const Ranges ranges(prefix[p.requests], Ranges::share_of(prefix[p.requests], (int)gridDim.x, p.pad_tiles));
  const int from = ranges.at(blockIdx.x, warp), to = ranges.at(blockIdx.x, warp + 1);
  bool merge = false;  // the CTA is inside one segment
  Segment cur = {};    // the segment of this warp's next tile, while it is known
  const int cta0 = ranges.at(blockIdx.x, 0);
  if (cta0 < ranges.total) {
    cur = segment_at<TK, ROWS>(p, prefix, cta0);
    merge = ranges.merged(blockIdx.x, cur.first, cur.first + cur.tiles);
    if (from < to && from >= cur.first + cur.tiles) cur = segment_at<TK, ROWS>(p, prefix, from);
  }
  const uint32_t ring = mbar::saddr(smem) + warp * C::STAGES * C::STAGE;
  const int BP = min(p.P, TK);              // tokens of a block in the ring
  // where this lane's keys, values and scales of 16-key block mt start in a stage
  const int kr = (g >> 1) + 4 * (g & 1);
  uint32_t k_code[MT], k_sca[MT], v_code[MT], v_sca[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const uint32_t blk = (uint32_t)(mt * 16 / BP) * L::bytes(BP), in = (mt * 16) & (BP - 1);
    k_code[mt] = blk + (in + kr) * L::CODE + t * (D == 64 ? 8 : 16);
    k_sca[mt] = blk + L::k_scale(BP) + (in + kr) * L::SCALE + t * (D == 64 ? 1 : 2);
    v_code[mt] = blk + L::v_code(BP) + (in + t) * L::CODE + g * (D / 16);
    v_sca[mt] = blk + L::v_scale(BP) + (in + t) * L::SCALE + (D == 64 ? g >> 1 : VG * g);
  }
  // this lane's 16 bytes of the value scales, for the NaN check: their key and place
  constexpr int KEYS16 = 16 / L::SCALE > 0 ? 16 / L::SCALE : 1;  // keys in 16 scale bytes
  const int nan_key = lane * KEYS16;
  const bool nan_lane = nan_key < TK;
  const uint32_t nan_at = nan_lane ? (uint32_t)(nan_key / BP) * L::bytes(BP) + L::v_scale(BP) + (nan_key & (BP - 1)) * L::SCALE : 0;

  JoinItem* items = reinterpret_cast<JoinItem*>(p.partial);
  float* pieces = p.partial + (int64_t)gridDim.x * kDecodeWarps * (sizeof(JoinItem) / 4);
  JoinItem* item = items + blockIdx.x * kDecodeWarps + warp;
  if (p.partial && lane == 0) item->rows = 0;

  // ---- feed the ring
  Feeder<D, TK> feed;
  int asked = from;  // tile of the line that is asked for next
  feed.left = 0;
  auto ask = [&]() {
    if (feed.left == 0) {
      const Segment s = asked < cur.first + cur.tiles ? cur : segment_at<TK, ROWS>(p, prefix, asked);
      feed.load(p, s.b, s.h, s.r.tile0 + asked - s.first, s.first + s.tiles - asked, s.r.end, lane);
    }
    const int st = (asked - from) % C::STAGES;
    feed.ask(p, ring + st * C::STAGE, mbar::saddr(&bars[warp][st]), lane);
    ++asked;
  };
  for (int s = 0; s < C::STAGES && asked < to; ++s) ask();

  bool dead = false;
  int tile = from;
  while (tile < to) {
    // ---- a segment: its rows' queries as the first product's second operand
    if (tile >= cur.first + cur.tiles) cur = segment_at<TK, ROWS>(p, prefix, tile);
    const Segment s = cur;
    const int rows = s.r.n * p.group;
    uint32_t qf[NT][STEPS][2];
    float f[NT][2];          // score -> log2 units, per column
    int hi[NT][2], lo[NT][2];  // visible keys of the column's row
    int all_hi = INT32_MAX, all_lo = 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = s.rb * ROWS + nt * 8 + g;
      const int qi = r / p.group, tok = s.r.t0 + qi;
      const bool real = r < rows && tok >= 0 && tok < p.tokens;
      const T* src = static_cast<const T*>(p.q) + (int64_t)(real ? tok : 0) * p.qts +
                     (int64_t)(s.h * p.group + (real ? r - qi * p.group : 0)) * p.qhs;
      float unscale = 1.f;
      uint4 v[WORDS];
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        const int d = D == 256 ? 32 * (t + 4 * (w >> 2)) + 8 * (w & 3) : t * (D / 4) + 8 * w;
        v[w] = real ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0, 0, 0, 0);
      }
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        uint32_t mx = 0;
#pragma unroll
        for (int w = 0; w < WORDS; ++w)
          mx = __vmaxu2(__vmaxu2(__vmaxu2(v[w].x & 0x7FFF7FFFu, v[w].y & 0x7FFF7FFFu),
                                 __vmaxu2(v[w].z & 0x7FFF7FFFu, v[w].w & 0x7FFF7FFFu)), mx);
        mx = max(mx & 0xFFFFu, mx >> 16);
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const int e = (int)(mx >> 7);  // the largest channel is below 2^(e - 126)
        // not finite: leave it; zero: nothing to scale
        const int k = e == 255 || mx == 0 ? 0 : min(14 + 126 - e, 126);
        const float up = __int_as_float((127 + k) << 23);
        unscale = __int_as_float((127 - k) << 23);
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
          uint32_t* u = reinterpret_cast<uint32_t*>(&v[w]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 x = unpack2<T>(u[i]);
            u[i] = pack2<__half>(x.x * up, x.y * up);
          }
        }
      }
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        qf[nt][2 * w][0] = v[w].x;
        qf[nt][2 * w][1] = v[w].y;
        qf[nt][2 * w + 1][0] = v[w].z;
        qf[nt][2 * w + 1][1] = v[w].w;
      }
      // this lane's columns are rows 2t, 2t + 1: their factors sit in lanes of those g
      const float fr = fmaxf(p.scale_log2 * unscale * p.cache.scales[s.h], 1.2e-38f);  // not 0: masked stays -inf
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        f[nt][j] = __shfl_sync(0xffffffffu, fr, (2 * t + j) * 4);
        const int c = s.rb * ROWS + nt * 8 + 2 * t + j;
        const int pos = s.r.pos0 + c / p.group;
        hi[nt][j] = c < rows ? min(pos + 1, s.r.end) : 0;
        lo[nt][j] = first_key(p, pos);
        if (c < rows) {
          all_hi = min(all_hi, hi[nt][j]);
          all_lo = max(all_lo, lo[nt][j]);
        }
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      all_hi = min(all_hi, __shfl_xor_sync(0xffffffffu, all_hi, o));
      all_lo = max(all_lo, __shfl_xor_sync(0xffffffffu, all_lo, o));
    }

    float o[NT][MI][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[nt][i][j] = 0.f;
    }
    uint32_t nan_seen = 0;
    const int piece0 = tile, stop = min(to, s.first + s.tiles);
    for (; tile < stop; ++tile) {
      const int st = (tile - from) % C::STAGES;
      if (!dead && !mbar::wait(mbar::saddr(&bars[warp][st]), ((tile - from) / C::STAGES) & 1, kWaitPolls)) {
        dead = true;
        if (lane == 0) atomicAdd(&g_timeouts, 1ull);
      }
      dead = __any_sync(0xffffffffu, dead);
      if (tile - s.first >= s.r.live) {  // padding
        if (asked < to && !dead) ask();
        continue;
      }
      const uint32_t sb = ring + st * C::STAGE;
      const int key0 = (s.r.tile0 + tile - s.first) * TK;

      // ---- S^T = K Q^T
      float sc[MT][NT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t w[2][WORDS], ks[2][WORDS / 2];
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const uint32_t code = sb + k_code[mt] + 8 * rr * L::CODE, sca = sb + k_sca[mt] + 8 * rr * L::SCALE;
          if constexpr (D == 64) {
            const uint2 v = lds_u64(code);
            w[rr][0] = v.x;
            w[rr][1] = v.y;
            ks[rr][0] = __byte_perm(fp8x2_to_f16x2<CEK_E4M3>(lds_u8(sca)), 0, 0x1010);
          } else {
#pragma unroll
            for (int j = 0; j < WORDS / 4; ++j) {
              const uint4 v = mbar::lds16(code + 64 * j);
              w[rr][4 * j] = v.x;
              w[rr][4 * j + 1] = v.y;
              w[rr][4 * j + 2] = v.z;
              w[rr][4 * j + 3] = v.w;
              const uint32_t two = fp8x2_to_f16x2<CEK_E4M3>(lds_u16(sca + 8 * j));
              ks[rr][2 * j] = __byte_perm(two, 0, 0x1010);
              ks[rr][2 * j + 1] = __byte_perm(two, 0, 0x3232);
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[mt][nt][j] = 0.f;
#pragma unroll
        for (int wd = 0; wd < WORDS; ++wd) {
          uint32_t x[2][4];
#pragma unroll
          for (int rr = 0; rr < 2; ++rr) {
            x[rr][0] = hmul2(e2m1x2_to_f16x2<0>(w[rr][wd]), ks[rr][wd / 2]);
            x[rr][1] = hmul2(e2m1x2_to_f16x2<1>(w[rr][wd]), ks[rr][wd / 2]);
            x[rr][2] = hmul2(e2m1x2_to_f16x2<2>(w[rr][wd]), ks[rr][wd / 2]);
            x[rr][3] = hmul2(e2m1x2_to_f16x2<3>(w[rr][wd]), ks[rr][wd / 2]);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816(sc[mt][nt], x[0][0], x[1][0], x[0][1], x[1][1], qf[nt][2 * wd][0], qf[nt][2 * wd][1]);
            mma16816(sc[mt][nt], x[0][2], x[1][2], x[0][3], x[1][3], qf[nt][2 * wd + 1][0], qf[nt][2 * wd + 1][1]);
          }
        }
      }

      // ---- softmax over the tile's keys (down the lanes of equal t)
      const bool inside = key0 + TK <= all_hi && key0 >= all_lo;
      float alpha[NT][2];
      bool moved = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float bias2[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (!inside) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int rr = 0; rr < 2; ++rr) {
                const int key = key0 + mt * 16 + rr * 8 + kr;
                if (key >= hi[nt][j] || key < lo[nt][j]) sc[mt][nt][2 * rr + j] = -INFINITY;
              }
          }
          float now = m[nt][j];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) now = max3(now, sc[mt][nt][j], sc[mt][nt][2 + j]);
          now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 4));
          now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 8));
          now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 16));
          const float bias = kShift - (now == -INFINITY ? 0.f : now * f[nt][j]);
          alpha[nt][j] = now == m[nt][j] ? 1.f : ex2((m[nt][j] - now) * f[nt][j]);
          moved |= now != m[nt][j];
          m[nt][j] = now;
          bias2[j] = bias;
        }
        // two columns an instruction
        const uint64_t ff = f32x2(f[nt][0], f[nt][1]), bb = f32x2(bias2[0], bias2[1]);
        uint64_t sum = 0;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int rr = 0; rr < 2; ++rr) {
            float &a = sc[mt][nt][2 * rr], &b = sc[mt][nt][2 * rr + 1];
            unpack_f32x2(fma_f32x2(f32x2(a, b), ff, bb), a, b);
            a = ex2(a);
            b = ex2(b);
            sum = add_f32x2(sum, f32x2(a, b));
          }
        float sa, sb2;
        unpack_f32x2(sum, sa, sb2);
        l[nt][0] = l[nt][0] * alpha[nt][0] + sa;
        l[nt][1] = l[nt][1] * alpha[nt][1] + sb2;
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < MI; ++i) {
            o[nt][i][0] *= alpha[nt][0];
            o[nt][i][1] *= alpha[nt][1];
            o[nt][i][2] *= alpha[nt][0];
            o[nt][i][3] *= alpha[nt][1];
          }
      }

      // ---- O^T += V^T P^T.  A slot without a token or behind a row counts p = 0;
      // a NaN scale must not turn that into NaN: it is 448 here, and the rows
      // that see its key get their NaN at the end of the segment.
      if (nan_lane && key0 + nan_key < s.r.end) {
        uint4 v = mbar::lds16(sb + nan_at);
        if (L::SCALE < 16 && key0 + nan_key + KEYS16 > s.r.end) {  // the last token is among the 16 bytes
          uint32_t* u = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key0 + nan_key + 4 * i / L::SCALE >= s.r.end) u[i] = 0;
        }
        nan_seen |= nan_bytes(v);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t pf[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          pf[nt][0] = movmatrix_t(pack2<__half>(sc[mt][nt][0], sc[mt][nt][1]));
          pf[nt][1] = movmatrix_t(pack2<__half>(sc[mt][nt][2], sc[mt][nt][3]));
        }
        uint32_t w[4][VW], vs[2][VG], sb8[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t code = sb + v_code[mt] + 4 * q * L::CODE, sca = sb + v_sca[mt] + 4 * q * L::SCALE;
          if constexpr (D == 64) {
            w[q][0] = lds_u32(code);
            sb8[q] = lds_u8(sca);
          } else if constexpr (D == 128) {
            const uint2 v = lds_u64(code);
            w[q][0] = v.x;
            w[q][1] = v.y;
            sb8[q] = lds_u8(sca);
          } else {
            const uint4 v = mbar::lds16(code);
            w[q][0] = v.x;
            w[q][1] = v.y;
            w[q][2] = v.z;
            w[q][3] = v.w;
            sb8[q] = lds_u16(sca);
          }
        }
        // scales of keys t, t + 4 and of t + 8, t + 12
#pragma unroll
        for (int j = 0; j < VG; ++j) {
          vs[0][j] = scales_no_nan(__byte_perm(sb8[0], sb8[1], j ? 0x0051 : 0x0040));
          vs[1][j] = scales_no_nan(__byte_perm(sb8[2], sb8[3], j ? 0x0051 : 0x0040));
        }
#pragma unroll
        for (int u = 0; u < VW; ++u) {
          // byte i: channels 8u + 2i (even) and 8u + 2i + 1 (odd) of two keys
          uint32_t even[2], odd[2];
#pragma unroll
          for (int k2 = 0; k2 < 2; ++k2) {
            const uint32_t a = w[2 * k2][u], b = w[2 * k2 + 1][u];
            even[k2] = (a & 0x0F0F0F0Fu) | ((b << 4) & 0xF0F0F0F0u);
            odd[k2] = ((a >> 4) & 0x0F0F0F0Fu) | (b & 0xF0F0F0F0u);
          }
          const uint32_t s0 = vs[0][VG == 2 ? u / 2 : 0], s1 = vs[1][VG == 2 ? u / 2 : 0];
#define CEK_KV4_PV(I)                                                                                            \
  {                                                                                                              \
    const uint32_t a0 = hmul2(e2m1x2_to_f16x2<I>(even[0]), s0), a1 = hmul2(e2m1x2_to_f16x2<I>(odd[0]), s0);      \
    const uint32_t a2 = hmul2(e2m1x2_to_f16x2<I>(even[1]), s1), a3 = hmul2(e2m1x2_to_f16x2<I>(odd[1]), s1);      \
    _Pragma("unroll") for (int nt = 0; nt < NT; ++nt)                                                            \
      mma16816(o[nt][4 * u + I], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);                                          \
  }
          CEK_KV4_PV(0)
          CEK_KV4_PV(1)
          CEK_KV4_PV(2)
          CEK_KV4_PV(3)
#undef CEK_KV4_PV
        }
      }
      __syncwarp();  // every lane has read the stage
      if (asked < to && !dead) ask();
    }

    // ---- end of the segment, or of this worker's part of it
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 4);
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 8);
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 16);
      }
    if (__any_sync(0xffffffffu, nan_seen != 0)) {
      // rare: look the keys' value scales up again, row by row
      const int k0 = (s.r.tile0 + piece0 - s.first) * TK, k1 = min(s.r.end, (s.r.tile0 + stop - s.first) * TK);
      for (int key = k0; key < k1; ++key) {
        const int id = min(max(p.table[(int64_t)s.b * p.table_stride + key / p.P], 0), p.cache.num_pages - 1);
        const uint8_t* sca = p.cache.data + (int64_t)id * p.cache.page_stride + (int64_t)s.h * p.cache.head_stride +
                             L::v_scale(p.P) + (key % p.P) * L::SCALE;
#pragma unroll
        for (int gr = 0; gr < VG; ++gr) {
          const bool nan = (sca[D == 64 ? g >> 1 : VG * g + gr] & 0x7F) == 0x7F;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (nan && key < hi[nt][j] && key >= lo[nt][j]) {
#pragma unroll
                for (int i = gr * (MI / VG); i < (gr + 1) * (MI / VG); ++i)
                  o[nt][i][j] = o[nt][i][2 + j] = __int_as_float(0x7fffffff);
              }
        }
      }
    }
    const bool mine = !merge && piece0 == s.first && stop == s.first + s.tiles;
    const float vf = p.cache.scales[p.cache.heads + s.h];
    if (p.partial && lane == 0 && piece0 == s.first && (merge ? s.first + s.tiles > ranges.at(blockIdx.x, kDecodeWarps) : !mine))
      *item = {s.first, s.first + s.tiles, ranges.total, ranges.share, s.r.t0, s.h, s.rb * ROWS, rows};
    // the ring is free once this warp's only segment is done: a merged piece goes there
    float* piece = merge ? reinterpret_cast<float*>(smem + warp * C::STAGES * C::STAGE)
                         : pieces + (int64_t)ranges.slot(blockIdx.x, warp, s.first, false) * (ROWS * (D + 2));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int col = nt * 8 + 2 * t + j, c = s.rb * ROWS + col;
        if (c >= rows) continue;
        if (mine) {
          const int qi = c / p.group, tok = s.r.t0 + qi;
          if (tok < 0 || tok >= p.tokens) continue;
          const float inv = l[nt][j] == 0.f ? 0.f : vf / l[nt][j];
          T* dst = static_cast<T*>(p.out) + (int64_t)tok * p.ots + (int64_t)(s.h * p.group + c - qi * p.group) * p.ohs +
                   g * (D / 8);
#pragma unroll
          for (int i = 0; i < MI; i += 4)
            *reinterpret_cast<uint4*>(dst + 2 * i) =
                make_uint4(pack2<T>(o[nt][i][j] * inv, o[nt][i][2 + j] * inv),
                           pack2<T>(o[nt][i + 1][j] * inv, o[nt][i + 1][2 + j] * inv),
                           pack2<T>(o[nt][i + 2][j] * inv, o[nt][i + 2][2 + j] * inv),
                           pack2<T>(o[nt][i + 3][j] * inv, o[nt][i + 3][2 + j] * inv));
        } else {
          if (g == 0) {
            piece[col] = m[nt][j] == -INFINITY ? -INFINITY : m[nt][j] * f[nt][j];
            piece[ROWS + col] = l[nt][j];
          }
          float* dst = piece + 2 * ROWS + col * D + g * (D / 8);
#pragma unroll
          for (int i = 0; i < MI; i += 2)
            *reinterpret_cast<float4*>(dst + 2 * i) =
                make_float4(o[nt][i][j], o[nt][i][2 + j], o[nt][i + 1][j], o[nt][i + 1][2 + j]);
        }
      }
  }
  // a wait gave up: the copies that are still in flight land before the block ends (bounded)
  if (dead)
    for (int a = max(from, asked - C::STAGES); a < asked; ++a)
      mbar::wait(mbar::saddr(&bars[warp][(a - from) % C::STAGES]), ((a - from) / C::STAGES) & 1, kWaitPolls);
  if (!merge) return;

  // ---- the four warps' pieces of the one segment, in the order of the keys
  const Segment s = cur;
  const int rows = s.r.n * p.group;
  const bool whole = ranges.at(blockIdx.x, 0) == s.first && ranges.at(blockIdx.x, kDecodeWarps) == s.first + s.tiles;
  __syncthreads();
  const float vf = p.cache.scales[p.cache.heads + s.h];
  float* piece = pieces + (int64_t)ranges.slot(blockIdx.x, 0, s.first, true) * (ROWS * (D + 2));
  for (int e = threadIdx.x; e < ROWS * (D / 8); e += kDecodeThreads) {
    const int col = e / (D / 8), d = e % (D / 8) * 8, c = s.rb * ROWS + col;
    if (c >= rows) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w)
      if (ranges.at(blockIdx.x, w) < ranges.at(blockIdx.x, w + 1))
        top = fmaxf(top, reinterpret_cast<const float*>(smem + w * C::STAGES * C::STAGE)[col]);
    const float base = top == -INFINITY ? 0.f : top;
    float l = 0.f, o[8] = {};
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) {
      if (ranges.at(blockIdx.x, w) >= ranges.at(blockIdx.x, w + 1)) continue;
      const float* q = reinterpret_cast<const float*>(smem + w * C::STAGES * C::STAGE);
      const float wt = ex2(q[col] - base);
      l += wt * q[ROWS + col];
      const float4 x = *reinterpret_cast<const float4*>(q + 2 * ROWS + col * D + d);
      const float4 y = *reinterpret_cast<const float4*>(q + 2 * ROWS + col * D + d + 4);
      o[0] += wt * x.x; o[1] += wt * x.y; o[2] += wt * x.z; o[3] += wt * x.w;
      o[4] += wt * y.x; o[5] += wt * y.y; o[6] += wt * y.z; o[7] += wt * y.w;
    }
    if (whole) {
      const int qi = c / p.group, tok = s.r.t0 + qi;
      if (tok < 0 || tok >= p.tokens) continue;
      const float inv = l == 0.f ? 0.f : vf / l;
      T* dst = static_cast<T*>(p.out) + (int64_t)tok * p.ots + (int64_t)(s.h * p.group + c - qi * p.group) * p.ohs + d;
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv),
                                                  pack2<T>(o[4] * inv, o[5] * inv), pack2<T>(o[6] * inv, o[7] * inv));
    } else {
      if (d == 0) {
        piece[col] = top;
        piece[ROWS + col] = l;
      }
      float4* dst = reinterpret_cast<float4*>(piece + 2 * ROWS + col * D + d);
      dst[0] = make_float4(o[0], o[1], o[2], o[3]);
      dst[1] = make_float4(o[4], o[5], o[6], o[7]);
    }
  }
}

// ---- joining the pieces of a segment --------------------------------------------
// CTA (c, y) joins the segments that decode CTA c's warps have left it.  Few
// pieces (a batch: what two neighbours share): CTA (c, 0) alone, a warp a row.
// Many (a long request): rows 2y and 2y + 1, four warps a row, each every fourth
// piece, then the four in order.  4 to 5 us, mostly the launch and two dependent
// reads (20 us before the pieces of a row were in flight together).
constexpr int kJoinWarps = 8, kJoinFew = 8, kJoinSub = 4, kJoinRows = kJoinWarps / kJoinSub;

template <int D>
struct Joined {
  float m = -INFINITY, l = 0.f, o[D / 32] = {};
  CEK_DEVICE void add(float mi, float li, const float (&oi)[D / 32]) {
    const float top = fmaxf(m, mi), base = top == -INFINITY ? 0.f : top, keep = ex2(m - base), wt = ex2(mi - base);
    l = l * keep + li * wt;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) o[e] = o[e] * keep + oi[e] * wt;
    m = top;
  }
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * kJoinWarps)
attn_join_kernel(const AttnParams p, int ctas) {
  constexpr int ROWS = 8 * NT, E = D / 32, SLOT = ROWS * (D + 2);
  __shared__ JoinItem items[kDecodeWarps];
  __shared__ float red[kJoinRows][kJoinSub][D], red_l[kJoinRows][kJoinSub], red_m[kJoinRows][kJoinSub];
  pdl_launch_dependents();
  pdl_wait();
  const int cta = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int WORDS = sizeof(JoinItem) / 4 * kDecodeWarps;
  const float* pieces = p.partial + (int64_t)ctas * WORDS;
  if (threadIdx.x < WORDS)
    reinterpret_cast<int*>(items)[threadIdx.x] = reinterpret_cast<const int*>(p.partial)[cta * WORDS + threadIdx.x];
  __syncthreads();
  for (int w = 0; w < kDecodeWarps; ++w) {
    const JoinItem s = items[w];
    if (s.rows == 0) continue;
    const Ranges ranges(s.total, s.share);
    // pieces: warps of the first CTA, whole CTAs, warps of the last CTA
    const int c1 = ranges.cta_of(s.end - 1);
    const bool one0 = ranges.merged(cta, s.first, s.end), one1 = ranges.merged(c1, s.first, s.end);
    const int n0 = one0 ? 1 : kDecodeWarps, mid = max(0, c1 - cta - 1);
    const int count = n0 + mid + (c1 > cta ? (one1 ? 1 : kDecodeWarps) : 0);
    const bool few = count <= kJoinFew;
    if (few && blockIdx.y > 0) continue;
    auto slot_at = [&](int k) -> int {
      if (k >= count) return -1;
      if (k >= n0 && k < n0 + mid) return ranges.slot(cta + 1 + k - n0, 0, s.first, true);
      const int kc = k < n0 ? cta : c1, kw = k < n0 ? k : k - n0 - mid;
      if (k < n0 ? one0 : one1) return ranges.slot(kc, 0, s.first, true);
      const int a = max(s.first, ranges.at(kc, kw)), b = min(s.end, ranges.at(kc, kw + 1));
      return a < b ? ranges.slot(kc, kw, s.first, false) : -1;
    };
    // pieces from, from + step, ... of a row, four in flight
    auto collect = [&](Joined<D>& j, int col, int from, int step) {
      constexpr int N = 4;
      for (int k0 = from; k0 < count; k0 += N * step) {
        float mi[N], li[N], oi[N][E];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int sl = slot_at(k0 + i * step);
          const float* q = pieces + (int64_t)max(sl, 0) * SLOT;
          mi[i] = sl >= 0 ? q[col] : -INFINITY;
          li[i] = sl >= 0 ? q[ROWS + col] : 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) oi[i][e] = sl >= 0 ? q[2 * ROWS + col * D + lane * E + e] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) j.add(mi[i], li[i], oi[i]);
      }
    };
    auto write = [&](const Joined<D>& j, int c) {
      const int qi = c / p.group, tok = s.t0 + qi;
      if (c >= s.rows || tok < 0 || tok >= p.tokens) return;
      const float inv = j.l == 0.f ? 0.f : p.cache.scales[p.cache.heads + s.h] / j.l;
      T* dst = static_cast<T*>(p.out) + (int64_t)tok * p.ots + (int64_t)(s.h * p.group + c - qi * p.group) * p.ohs + lane * E;
      uint32_t u[E / 2];
#pragma unroll
      for (int e = 0; e < E / 2; ++e) u[e] = pack2<T>(j.o[2 * e] * inv, j.o[2 * e + 1] * inv);
      if constexpr (E == 2) *reinterpret_cast<uint32_t*>(dst) = u[0];
      else if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(u[0], u[1]);
      else *reinterpret_cast<uint4*>(dst) = make_uint4(u[0], u[1], u[2], u[3]);
    };
    if (few) {
      for (int col = warp; col < ROWS && s.row0 + col < s.rows; col += kJoinWarps) {
        Joined<D> j;
        collect(j, col, 0, 1);
        write(j, s.row0 + col);
      }
      continue;
    }
    const int jr = warp / kJoinSub, sub = warp % kJoinSub, col = blockIdx.y * kJoinRows + jr;
    Joined<D> j;
    if (s.row0 + col < s.rows) collect(j, col, sub, kJoinSub);
#pragma unroll
    for (int e = 0; e < E; ++e) red[jr][sub][lane * E + e] = j.o[e];
    if (lane == 0) {
      red_l[jr][sub] = j.l;
      red_m[jr][sub] = j.m;
    }
    __syncthreads();
    if (sub == 0) {
#pragma unroll
      for (int i = 1; i < kJoinSub; ++i) {
        float oi[E];
#pragma unroll
        for (int e = 0; e < E; ++e) oi[e] = red[jr][i][lane * E + e];
        j.add(red_m[jr][i], red_l[jr][i], oi);
      }
      write(j, s.row0 + col);
    }
    __syncthreads();
  }
}

}  // namespace kv4
}  // namespace cek

// ---- host side -------------------------------------------------------------------
namespace {
using namespace cek::kv4;

// Rows of a kv head that the decode kernel takes.  At 17 to 32 rows (two passes of
// 16) it beats the tensor-core kernel for narrow heads: 16 requests of 5 rows on
// 16/4 heads of 64, 4000 keys, 24.6 us against 28.6; one of 4 tokens on 64/8 heads
// of 128, 500 keys, 10.7 against 12.8.  At 256 channels two n8 blocks of rows do
// not fit its registers: 16 rows on 500 keys 21.5 us against 16.4.
inline int64_t decode_rows(int64_t d) { return d == 256 ? 8 : 32; }

// Keys of a request and rows of its kv head: 32-bit numbers with room for a tile or a row block behind them.
constexpr int64_t kMaxKeys = INT32_MAX - 127, kMaxRows = INT32_MAX - 1023;

struct DecodePlan {
  int nt, tile_keys, ctas;
  int pad;              // tiles of a segment where all are short, else 0
  size_t smem;
  bool join;            // some segment may be in several pieces
  int64_t partial_bytes;
};

template <int D, int NT>
DecodePlan plan_decode_dn(int64_t requests, int64_t heads, int64_t group, int64_t max_q, int64_t max_seq) {
  using C = DecodeCfg<D, NT>;
  DecodePlan d;
  d.nt = NT;
  d.tile_keys = C::TK;
  const int64_t req = std::min<int64_t>(requests, kMaxRequests);
  const int64_t segments = req * heads * ((max_q * group + 8 * NT - 1) / (8 * NT));
  const int64_t tiles = std::max<int64_t>(1, (max_seq + C::TK - 1) / C::TK);
  d.smem = (size_t)C::RING + sizeof(int32_t) * (req + 1);
  const int per_sm = (int)std::min<int64_t>(C::PER_SM, 233472 / (d.smem + 1024 + 512));  // 228 KB an SM, 1 KB a CTA reserved
  const int64_t most = (int64_t)std::max(1, per_sm) * cek_host::sm_count();
  // (A window is not counted: its few tiles behind a long bound are cut all the same.)
  // A cut costs a second launch, 4 to 5 us: with a CTA for every segment, two tiles a warp
  // (another 1.3 us) are cheaper; otherwise a warp takes whole segments of up to four.
  d.pad = tiles <= (segments <= most ? 2 : 1) * kDecodeWarps ? (int)tiles : 0;
  d.ctas = (int)std::min(most, segments >= most ? most : segments * (d.pad ? 1 : (tiles + kDecodeWarps - 1) / kDecodeWarps));
  d.join = d.pad == 0;
  d.partial_bytes = d.join ? (int64_t)kDecodeWarps * d.ctas * (sizeof(JoinItem) + 2 * 8 * NT * (D + 2) * sizeof(float)) : 0;
  return d;
}
template <int D>
DecodePlan plan_decode_d(int64_t requests, int64_t heads, int64_t group, int64_t max_q, int64_t max_seq) {
  if constexpr (D < 256)
    if (max_q * group > 8) return plan_decode_dn<D, 2>(requests, heads, group, max_q, max_seq);
  return plan_decode_dn<D, 1>(requests, heads, group, max_q, max_seq);
}
DecodePlan plan_decode(int64_t d, int64_t requests, int64_t heads, int64_t group, int64_t max_q, int64_t max_seq) {
  return d == 64    ? plan_decode_d<64>(requests, heads, group, max_q, max_seq)
         : d == 128 ? plan_decode_d<128>(requests, heads, group, max_q, max_seq)
                    : plan_decode_d<256>(requests, heads, group, max_q, max_seq);
}

// Requests of one launch: their prefix sums sit in shared memory, and the line of their tiles
// is counted in 32 bits with room for a product by the warps of a CTA.  0: one has too many tiles.
int64_t decode_requests(const AttnParams& p, const DecodePlan& d) {
  const int64_t keys = std::min(p.max_seq, p.key_limit);
  const int64_t tiles = std::max<int64_t>(std::max(1, d.pad), (keys + d.tile_keys - 1) / d.tile_keys);
  const int64_t blocks = ((int64_t)p.max_q * p.group + 8 * d.nt - 1) / (8 * d.nt);
  return std::min<int64_t>(kMaxRequests, INT32_MAX / kDecodeWarps / (tiles * p.cache.heads * blocks));
}

template <typename T, int D, int NT>
int launch_decode(const AttnParams& p, const DecodePlan& d, cudaStream_t st) {
  static cek_host::DeviceSlots attr;
  if (!cek_host::ensure_smem_attr(attr, attn_decode_kernel<T, D, NT>, DecodeCfg<D, NT>::RING + 4 * (kMaxRequests + 1)))
    return CEK_ERR_LAUNCH;
  int s = cek_host::launch_pdl(attn_decode_kernel<T, D, NT>, dim3(d.ctas), dim3(kDecodeThreads), d.smem, st, p);
  if (s != CEK_OK || !d.join) return s;
  return cek_host::launch_pdl(attn_join_kernel<T, D, NT>, dim3(d.ctas, 8 * NT / kJoinRows),
                              dim3(32 * kJoinWarps), 0, st, p, d.ctas);
}
template <typename T>
int launch_decode_t(int64_t dim, const AttnParams& p, const DecodePlan& d, cudaStream_t st) {
  if (dim == 64) return d.nt == 1 ? launch_decode<T, 64, 1>(p, d, st) : launch_decode<T, 64, 2>(p, d, st);
  if (dim == 128) return d.nt == 1 ? launch_decode<T, 128, 1>(p, d, st) : launch_decode<T, 128, 2>(p, d, st);
  return launch_decode<T, 256, 1>(p, d, st);
}
}  // namespace

extern "C" int64_t cek_kv4_attention_workspace_bytes(int64_t requests, int64_t tokens, int64_t q_heads,
                                                     int64_t kv_heads, int64_t head_dim, int64_t max_query_len,
                                                     int64_t max_seq_len) {
  if (requests <= 0 || tokens <= 0 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads || max_query_len <= 0 ||
      max_seq_len <= 0 || !cek_host::kv4_head_dim(head_dim))
    return 0;
  const int64_t group = q_heads / kv_heads, max_q = std::min(max_query_len, tokens);
  if (max_q * group <= decode_rows(head_dim))
    return plan_decode(head_dim, requests, kv_heads, group, max_q, max_seq_len).partial_bytes;
  return cek::kv4::prefill_workspace(head_dim, requests, tokens, kv_heads, group, max_q, max_seq_len);
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
      q_heads % cache->kv_heads || q_heads > 65535 || table_width < 0 || table_width > kMaxKeys / cache->page_size ||
      table_stride < table_width || max_query_len < 0 || max_seq_len < 0 || max_query_len > INT32_MAX ||
      max_seq_len > INT32_MAX || window < 0 || window > INT32_MAX)
    return CEK_ERR_INVALID_ARG;
  if (std::min(max_query_len, tokens) * (q_heads / cache->kv_heads) > kMaxRows) return CEK_ERR_INVALID_ARG;
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
  p.group = (int)(q_heads / cache->kv_heads);
  p.P = (int)cache->page_size;
  while ((1 << p.page_shift) < p.P) ++p.page_shift;
  p.max_q = (int)std::min(max_query_len, tokens);
  p.max_seq = (int)max_seq_len;
  p.key_limit = (int)(table_width * cache->page_size);
  p.window = (int)window;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  if (p.max_q * p.group <= decode_rows(cache->head_dim)) {
    const DecodePlan d = plan_decode(cache->head_dim, requests, cache->kv_heads, p.group, p.max_q, max_seq_len);
    if (workspace_bytes < d.partial_bytes || (d.partial_bytes > 0 && !workspace)) return CEK_ERR_INVALID_ARG;
    if (d.partial_bytes > 0 && !cek_host::aligned16(workspace)) return CEK_ERR_ALIGNMENT;
    p.partial = d.join ? static_cast<float*>(workspace) : nullptr;
    p.pad_tiles = d.pad;
    const int64_t part = decode_requests(p, d);
    if (part == 0) return CEK_ERR_INVALID_ARG;
    int rc = CEK_OK;
    for (int64_t b = 0; b < requests && rc == CEK_OK; b += part) {
      p.requests = (int)std::min(part, requests - b);
      p.table = block_table + b * table_stride;
      p.query_start = query_start + b;
      p.seq_lens = seq_lens + b;
      rc = dtype == CEK_F16 ? launch_decode_t<__half>(cache->head_dim, p, d, static_cast<cudaStream_t>(stream))
                            : launch_decode_t<__nv_bfloat16>(cache->head_dim, p, d, static_cast<cudaStream_t>(stream));
    }
    return rc;
  }
  const int64_t need = cek::kv4::prefill_workspace(cache->head_dim, requests, tokens, cache->kv_heads, p.group,
                                                        p.max_q, max_seq_len);
  if (workspace_bytes < need || (need > 0 && !workspace)) return CEK_ERR_INVALID_ARG;
  if (need > 0 && !cek_host::aligned16(workspace)) return CEK_ERR_ALIGNMENT;
  p.partial = static_cast<float*>(workspace);
  return cek::kv4::prefill_launch(dtype, cache->head_dim, p, max_seq_len, static_cast<cudaStream_t>(stream));
}

extern "C" int cek_kv4_timeouts(uint64_t* count) {
  if (!count) return CEK_ERR_INVALID_ARG;
  unsigned long long a = 0, b = 0;
  if (cudaMemcpyFromSymbol(&a, cek::kv4::g_timeouts, sizeof(a)) != cudaSuccess || !cek::kv4::prefill_timeouts(&b))
    return CEK_ERR_LAUNCH;
  *count = a + b;
  return CEK_OK;
}
