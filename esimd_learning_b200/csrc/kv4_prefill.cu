// kv4_prefill.cu — attention over the paged 4-bit cache for many rows a
// request (prompts, chunks): cek_kv4_attention's tcgen05 path.
//
// A CTA takes NQ x 128 rows (query token x head of the kv head's group) and the
// tiles of TK keys that any of them sees.  16 warps:
//  * softmax (one warpgroup per 128 rows, a thread a row): stages Q in shared
//    memory, then per tile reads S from tensor memory, keeps the
//    running maximum and sum, and writes P (fp16) over S;
//  * converters: turn the codes of a page into the fp16 operands, exactly
//    (kv4.cuh), straight into the 128-byte-swizzled layout that the matrix unit
//    reads; a ring of slots K(j), V(j), K(j+1), ...
//  * one warp copies pages (a bulk copy per page, keys and values apart) into a raw
//    ring, in the order in which the converters free it;
//  * one warp issues the matrix instructions: S = Q K^T with both operands in
//    shared memory, O += P V with P in tensor memory and V read with keys as
//    the strided dimension, so V needs no transpose.
// With NQ = 2 the two row blocks take turns: while one's S is in softmax the
// other's products run.  D = 256 fills tensor memory with one O, so NQ = 1 and
// the tiles take turns instead (S double-buffered).
//
// With work for every SM, D >= 128 runs on pairs of CTAs (CG = 2,
// cta_group::2): a product has 256 rows, each CTA keeps and reads half of K's
// rows and of V's channels, and so converts half.  Alone, the first product is
// bound by its operands (128 bytes a cycle of shared memory, all of it) and
// takes 920 cycles instead of 512 beside the converters.
//
// Per 256 rows x 128 keys at D = 128 a CTA needs 2048 cycles of matrix unit,
// 2048 of exp2 (16 a cycle) and, in a pair, ~1500 of shared memory.  It takes
// ~3500: a row block's softmax (2000) and its products (1024) follow each other,
// and each hand-over costs a few hundred cycles; two row blocks hide a part of it.
// 8192 tokens of 64/8 heads of 128 from an empty cache: 1085 us, 1010 TFLOP/s.  Six
// ragged chunks of 16/4 heads of 256 with a window of 1024: 147 us, 557 TFLOP/s;
// there an item starts for 6 us and ends for 3 of its 27.
//
// The output is rescaled only when a row's maximum has grown by more than
// 2^kLazy since the last time: P is at most 2^(kShift + kLazy) = 2^14 then,
// inside fp16, and fp16 keeps P's full precision down to 2^-20 of the maximum.
// Every wait is bounded; one that gives up is counted (cek_kv4_timeouts), the
// CTA drains its copies and matrix instructions, frees its tensor memory and
// returns.
#include "kv4_attention.cuh"

#include <algorithm>
#include <type_traits>

namespace cek {
namespace kv4 {

__device__ unsigned long long g_timeouts_prefill;

namespace pf {

constexpr float kShift = 6.f, kLazy = 8.f;
constexpr int kThreads = 512;
constexpr uint32_t kPolls = 1u << 24;
constexpr int kSmem = 226 * 1024;  // dynamic shared memory of a CTA at most

// CG CTAs share their K and V (a cluster).
template <int D, int NQ, int CG>
struct Cfg {
  // 128 keys a tile: products of 64 columns take the matrix unit as long as ones of 128.  One
  // CTA's K and V of 256 channels leave room for 64.
  static constexpr int TK = D == 256 && CG == 1 ? 64 : 128;
  static constexpr int ROWS = NQ * 128;                   // of a CTA; an item has CG of them
  static constexpr int Q_BYTES = ROWS * D * 2, SLOT = TK * D * 2 / CG;
  static constexpr int RAW = Layout<D>::v_code(TK);       // a raw stage: a tile's keys or values
  static constexpr int SLOTS = 4;                         // converted K and V tiles
  // raw stages: what is left, 16 at most
  static constexpr int RAW_ROOM = (kSmem - 1024 - Q_BYTES - SLOTS * SLOT) / RAW, RAWS = RAW_ROOM < 16 ? RAW_ROOM : 16;
  static constexpr int SMEM = Q_BYTES + SLOTS * SLOT + RAWS * RAW + 1024;
  static constexpr int CONV_WARPS = NQ == 2 ? 4 : 8;      // warps 8..11, or 4..11
  static constexpr int O_COL = 256;
  static constexpr uint32_t IDESC_QK = (1u << 4) | (uint32_t(TK >> 3) << 17) | (uint32_t(8 * CG) << 24);
  // bit 16: B (V) has its N dimension contiguous
  static constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 16) | (uint32_t(D >> 3) << 17) | (uint32_t(8 * CG) << 24);
};

CEK_DEVICE bool wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  for (uint32_t i = 0; i < kPolls; ++i) {
    if (mbar::try_wait(bar, parity)) return true;
    if ((i & 1023u) == 1023u && *abort_flag) return false;
  }
  *abort_flag = 1;
  atomicAdd(&g_timeouts_prefill, 1ull);
  return false;
}
// The same by a whole warp, with one answer for all of it.
CEK_DEVICE bool wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, wait(bar, parity, abort_flag));
}
CEK_DEVICE uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
CEK_DEVICE void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
CEK_DEVICE void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Arrives on `bar` of every CTA of the group when the products issued so far are done.
template <int CG>
CEK_DEVICE void commit(uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"((uint16_t)3)
                 : "memory");
}
// Arrives on the leading CTA's `bar` (this CTA's, where it is alone).  What the
// arrival announces is complete before it: converted tiles by fence.proxy.async,
// P by tcgen05.wait::st and fence::before_thread_sync.  It need not order more
// (release at cluster scope cost some 900 cycles each time, twice the products).
template <int CG>
CEK_DEVICE void arrive_lead(uint32_t bar) {
  if constexpr (CG == 1)
    mbar::arrive(bar);
  else
    asm volatile(
        "{ .reg .b32 r; mapa.shared::cluster.u32 r, %0, 0; mbarrier.arrive.shared::cluster.b64 _, [r]; }" ::"r"(bar)
        : "memory");
}
// Stores to the same place in every CTA of the group.
template <int CG>
CEK_DEVICE void store_all(uint32_t addr, uint32_t v) {
#pragma unroll
  for (int r = 0; r < CG; ++r)
    asm volatile("{ .reg .b32 a; mapa.shared::cluster.u32 a, %0, %1; st.shared::cluster.u32 [a], %2; }" ::"r"(addr), "r"(r), "r"(v)
                 : "memory");
}
// A barrier of all threads of the group, memory included.
template <int CG>
CEK_DEVICE void sync_group() {
  if constexpr (CG == 1)
    __syncthreads();
  else
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Shared-memory descriptor, 128-byte swizzle, 8-row groups 1024 bytes apart;
// `lead` is the distance of 64-element blocks where those are contiguous (V).
CEK_DEVICE uint64_t desc(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lead >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
template <int CG>
CEK_DEVICE void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (CG == 1)
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
  else
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
template <int CG>
CEK_DEVICE void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (CG == 1)
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
  else
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
// One lane of a converged warp.  The warp stays together around it, so that
// addresses and descriptors are warp-uniform for the compiler: issued from a
// branch on the lane number the matrix instructions took twice as long.
CEK_DEVICE bool elect() {
  uint32_t p;
  asm volatile("{ .reg .pred e; elect.sync _|e, 0xffffffff; selp.u32 %0, 1, 0, e; }" : "=r"(p));
  return p != 0;
}
CEK_DEVICE void tmem_ld32(uint32_t addr, float* r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(addr));
}
CEK_DEVICE void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
CEK_DEVICE void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
CEK_DEVICE void tmem_st16(uint32_t addr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]) : "memory");
}
CEK_DEVICE void sts16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
CEK_DEVICE void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The rows and tiles of one CTA.
struct Item {
  int b, h, rb, split;
  Request r;
  int rows;            // of the request's kv head
  int tile0, tiles;    // of this split
  int limit;           // no row of the block sees a key at or past it
};
// The block's item; false: there is none.  The whole block calls it.  Row blocks of
// the longest request are `row_blocks`: items are counted as if every request had
// as many, the longest ranges first.  With row_blocks = 0 (a few prompts among many
// short requests, where most of those would be empty) they are counted one by one,
// request by request.
template <int TK, int ROWS, int CG>
CEK_DEVICE bool item_of(const AttnParams& p, int row_blocks, int splits, Item& it) {
  uint32_t id = blockIdx.x / CG;
  const uint32_t sp = id / (uint32_t)splits;
  it.split = (int)(id - sp * (uint32_t)splits);
  id = sp / (uint32_t)p.cache.heads;
  it.h = (int)(sp - id * (uint32_t)p.cache.heads);
  if (row_blocks > 0) {
    const uint32_t up = id / (uint32_t)p.requests;
    it.b = (int)(id - up * (uint32_t)p.requests);
    it.rb = row_blocks - 1 - (int)up;
  } else {
    __shared__ int sums[kThreads / 32], found[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) found[0] = -1;
    int64_t before = 0;
    for (int b0 = 0; b0 < p.requests && before <= id; b0 += kThreads) {
      const int b = b0 + tid;
      int n = 0;
      if (b < p.requests) {
        n = min(max(p.query_start[b + 1] - p.query_start[b], 0), p.max_q);
        n = (int)(((int64_t)n * p.group + ROWS - 1) / ROWS);
      }
      int s = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += v;
      }
      __syncthreads();
      if (lane == 31) sums[warp] = s;
      __syncthreads();
      int64_t first = before + s - n;
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) first += sums[w];
        before += sums[w];
      }
      if (id >= first && id < first + n) {
        found[0] = b;
        found[1] = n - 1 - (int)(id - first);
      }
    }
    __syncthreads();
    if (found[0] < 0) return false;
    it.b = found[0];
    it.rb = found[1];
  }
  it.r = request_of<TK>(p, it.b);
  it.rows = it.r.n * p.group;
  if (it.rb * ROWS >= it.rows) return false;
  const int last = min(it.rows, (it.rb + 1) * ROWS) - 1;
  const int lo = first_key(p, it.r.pos0 + it.rb * ROWS / p.group);
  it.limit = min(it.r.pos0 + last / p.group + 1, it.r.end);
  const int t0 = lo / TK, n = it.limit > lo ? (it.limit + TK - 1) / TK - t0 : 0;
  const int a = (int)((int64_t)n * it.split / splits), z = (int)((int64_t)n * (it.split + 1) / splits);
  it.tile0 = t0 + a;
  it.tiles = z - a;
  return true;
}

template <typename T, int D, int NQ, int CG>
__global__ void __launch_bounds__(kThreads, 1)
attn_prefill_kernel(const AttnParams p, int row_blocks, int splits) {
  using C = Cfg<D, NQ, CG>;
  using L = Layout<D>;
  constexpr int TK = C::TK, ROWS = C::ROWS, GP = D / 16;
  static_assert(CG == 1 || D >= 128, "a pair halves V by 64 channels at least");
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sbase = (mbar::saddr(smem_raw) + 1023u) & ~1023u;
  const uint32_t s_q = sbase, s_kv = sbase + C::Q_BYTES, s_rw = s_kv + C::SLOTS * C::SLOT;
  constexpr int kRaw = C::RAWS, kSlots = C::SLOTS;
  __shared__ __align__(8) uint64_t raw_full[kRaw], raw_empty[kRaw], kv_full[kSlots], kv_empty[kSlots], s_full[2], p_full[2], o_done[2],
      q_full, drain;
  __shared__ float row_unscale[ROWS];
  __shared__ uint32_t tmem_sh;
  __shared__ volatile int abort_flag;
  __shared__ volatile uint32_t nan_seen;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar::init(mbar::saddr(&kv_full[i]), CG * C::CONV_WARPS);
      mbar::init(mbar::saddr(&kv_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar::init(mbar::saddr(&s_full[i]), 1);
      mbar::init(mbar::saddr(&p_full[i]), CG * 4);
      mbar::init(mbar::saddr(&o_done[i]), 1);
    }
    mbar::init(mbar::saddr(&q_full), CG * 4 * NQ);
    mbar::init(mbar::saddr(&drain), 1);
    abort_flag = 0;
    nan_seen = 0;
    mbar::fence_init();
  }
  pdl_wait();
  Item it;
  if (!item_of<TK, CG * ROWS, CG>(p, row_blocks, splits, it)) return;  // the whole group
  const uint32_t rank = CG == 1 ? 0 : cta_rank();
  const int n = it.tiles;
  const bool soft = warp < 4 * NQ;

  // what a softmax thread keeps until the end
  const int x = NQ == 2 ? warp >> 2 : 0;                       // its stream of row blocks
  const int rr = (warp & 3) * 32 + lane;                       // its row of the block
  const int row = (it.rb * CG + (int)rank) * ROWS + x * 128 + rr;
  const int qi = row / p.group, tok = it.r.t0 + qi, head = it.h * p.group + row - qi * p.group;
  const bool real = soft && row < it.rows && tok >= 0 && tok < p.tokens;
  const int pos = it.r.pos0 + qi;
  const int hi = row < it.rows ? min(pos + 1, it.r.end) : 0, lo = first_key(p, pos);

  constexpr int LPR = D / 8, RPI = 32 / LPR;  // lanes of a row of Q or of the output, rows at a time
  const int ch = lane % LPR;

  // Q and the first pages are on their way before the group meets (with plain loads the
  // barrier would wait for Q).  Q: the warp's 32 rows, whole rows at a time; 16-byte
  // chunk ch of 64-channel block cb goes to ch ^ (row & 7); rows that are not there are 0.
  auto q_at = [&](int i) {
    const int r = (warp & 3) * 32 + i * RPI + lane / LPR;
    return s_q + x * (128 * D * 2) + (ch >> 3) * (128 * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
  };
  if (soft) {
    const int64_t own = real ? (int64_t)tok * p.qts + (int64_t)head * p.qhs : -1;
#pragma unroll 8
    for (int i = 0; i < LPR; ++i) {
      const int64_t at = __shfl_sync(0xffffffffu, own, i * RPI + lane / LPR);
      const T* src = static_cast<const T*>(p.q) + max(at, (int64_t)0) + ch * 8;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(q_at(i)), "l"(src), "r"(at >= 0 ? 16 : 0) : "memory");
    }
  }
  Feeder<D, TK> feed;
  int pages = 0;  // stages asked for
  auto ask = [&](int i) {
    const int key0 = (it.tile0 + (i >> 1)) * TK;
    if ((i & 1) == 0) feed.look(p, key0, lane);
    const uint32_t dst = s_rw + (i % kRaw) * C::RAW, bar = mbar::saddr(&raw_full[i % kRaw]);
    if ((i & 1) == 0) feed.template ask_part<TK / CG>(p, dst, bar, lane, key0 + (int)rank * (TK / CG), 0);
    else feed.template ask_part<TK>(p, dst, bar, lane, key0, 1);
  };
  if (warp == 13) {
    if (lane == 0) {
      for (int i = 0; i < kRaw; ++i) {
        mbar::init(mbar::saddr(&raw_full[i]), 1);
        mbar::init(mbar::saddr(&raw_empty[i]), C::CONV_WARPS);
      }
      mbar::fence_init();
    }
    __syncwarp();
    if (n > 0) feed.load(p, it.b, it.h, it.tile0, n, it.limit, lane);
    for (; pages < min(2 * n, min(2, kRaw)); ++pages) ask(pages);  // one tile: more would hold up the others
  }
  if (warp == 12) {
    if constexpr (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(mbar::saddr(&tmem_sh)), "r"(512));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(mbar::saddr(&tmem_sh)), "r"(512));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
  }
  fence_before();
  sync_group<CG>();
  fence_after();
  const uint32_t tmem = tmem_sh;
  const uint32_t tm_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  float m = -INFINITY, l = 0.f, c = 0.f, vf = 0.f;

  if (soft) {
    if constexpr (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    asm volatile("cp.async.wait_all;" ::: "memory");
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      // as in the decode kernel: each row by a power of two, exactly, into fp16's range; a lane
      // converts the chunks that it has copied
#pragma unroll 1
      for (int i0 = 0; i0 < LPR; i0 += 8) {  // eight rows' chains side by side
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = mbar::lds16(q_at(i0 + i));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t mx = __vmaxu2(__vmaxu2(v[i].x & 0x7FFF7FFFu, v[i].y & 0x7FFF7FFFu),
                                 __vmaxu2(v[i].z & 0x7FFF7FFFu, v[i].w & 0x7FFF7FFFu));
          mx = max(mx & 0xFFFFu, mx >> 16);
          mx = __reduce_max_sync(LPR == 32 ? 0xffffffffu : ((1u << (LPR & 31)) - 1) << (lane / LPR * LPR), mx);
          const int e = (int)(mx >> 7);
          const int k = e == 255 || mx == 0 ? 0 : min(14 + 126 - e, 126);
          const float up = __int_as_float((127 + k) << 23);
          if (ch == 0) row_unscale[x * 128 + (warp & 3) * 32 + (i0 + i) * RPI + lane / LPR] = __int_as_float((127 - k) << 23);
          uint32_t* u = reinterpret_cast<uint32_t*>(&v[i]);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float2 f = unpack2<T>(u[q]);
            u[q] = pack2<__half>(f.x * up, f.y * up);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sts16(q_at(i0 + i), v[i].x, v[i].y, v[i].z, v[i].w);
      }
    }
    proxy_fence();
    __syncwarp();
    if (lane == 0) arrive_lead<CG>(mbar::saddr(&q_full));
    vf = p.cache.scales[p.cache.heads + it.h];
    const float unscale = std::is_same<T, __nv_bfloat16>::value ? row_unscale[x * 128 + rr] : 1.f;
    // score -> log2 units; not zero, so that a masked -inf stays -inf
    c = fmaxf(p.scale_log2 * unscale * p.cache.scales[it.h], 1.2e-38f);
    int whi = hi, wlo = lo;  // keys that every row of the warp sees
    if (row >= it.rows) whi = INT32_MAX, wlo = 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      whi = min(whi, __shfl_xor_sync(0xffffffffu, whi, o));
      wlo = max(wlo, __shfl_xor_sync(0xffffffffu, wlo, o));
    }
    const uint32_t tm_o = tm_lane + C::O_COL + x * D;

    for (int j = 0; j < n; ++j) {
      const int buf = NQ == 2 ? x : j & 1;
      const uint32_t par = NQ == 2 ? j & 1 : (j >> 1) & 1;
      if (!wait_warp(mbar::saddr(&s_full[buf]), par, &abort_flag)) break;
      fence_after();
      const uint32_t tm_s = tm_lane + buf * 128;
      float s[TK];
#pragma unroll
      for (int i = 0; i < TK; i += 32) tmem_ld32(tm_s + i, s + i);
      tmem_ld_wait();
      const int key0 = (it.tile0 + j) * TK;
      if (key0 < wlo || key0 + TK > whi) {
#pragma unroll
        for (int i = 0; i < TK; ++i)
          if (key0 + i < lo || key0 + i >= hi) s[i] = -INFINITY;
      }
      float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int i = 4; i < TK - 4; i += 8)
#pragma unroll
        for (int q = 0; q < 4; ++q) top[q] = max3(top[q], s[i + 2 * q], s[i + 2 * q + 1]);
#pragma unroll
      for (int q = 0; q < 4; ++q) top[q] = fmaxf(top[q], s[TK - 4 + q]);
      const float mx = fmaxf(max3(top[0], top[1], top[2]), top[3]);
      const float now = fmaxf(m, mx);
      // (a - b) * c of equal infinities is NaN: not a reason to rescale
      const bool grow = (now - m) * c > kLazy;
      if (__any_sync(0xffffffffu, grow)) {
        if (j > 0) {
          if (!wait_warp(mbar::saddr(&o_done[x]), (j - 1) & 1, &abort_flag)) break;
          fence_after();
          const float alpha = grow ? ex2((m - now) * c) : 1.f;
          l *= alpha;
#pragma unroll 1
          for (int i = 0; i < D; i += 32) {
            float o[32];
            tmem_ld32(tm_o + i, o);
            tmem_ld_wait();
#pragma unroll
            for (int q = 0; q < 32; ++q) o[q] *= alpha;
            tmem_st16(tm_o + i, reinterpret_cast<uint32_t*>(o));
            tmem_st16(tm_o + i + 16, reinterpret_cast<uint32_t*>(o) + 16);
          }
          tmem_st_wait();
        }
        if (grow) m = now;
      }
      const float bias = kShift - (m == -INFINITY ? 0.f : m * c);
      const uint64_t c2 = f32x2(c, c), bias2 = f32x2(bias, bias);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < TK; i += 32) {
        uint32_t u[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          float a, b;
          unpack_f32x2(fma_f32x2(f32x2(s[i + 2 * q], s[i + 2 * q + 1]), c2, bias2), a, b);
          a = ex2(a);
          b = ex2(b);
          sum[q & 1] = add_f32x2(sum[q & 1], f32x2(a, b));
          u[q] = pack2<__half>(a, b);
        }
        tmem_st16(tm_s + i / 2, u);
      }
      float la, lb;
      unpack_f32x2(add_f32x2(sum[0], sum[1]), la, lb);
      l += la + lb;
      tmem_st_wait();
      fence_before();
      __syncwarp();
      if (lane == 0) arrive_lead<CG>(mbar::saddr(&p_full[buf]));
    }
    if (n > 0) wait(mbar::saddr(&o_done[x]), (n - 1) & 1, &abort_flag);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp < 12) {
      // ---- converters: thread items are 16-channel groups of a key, the same
      // places in every tile.  Of a pair each CTA converts its half of the second
      // operand's columns: half the keys of K, half the channels of V.
      constexpr int NTHR = C::CONV_WARPS * 32, ITEMS = TK * GP / (NTHR * CG);
      const int ct = threadIdx.x - (12 - C::CONV_WARPS) * 32;
      struct Places {
        uint32_t from[ITEMS], from_s[ITEMS], to, flip;
        int row0;
      };
      // KEYS keys, GR groups from group g0 on
      auto places = [&](auto keys, auto groups, int g0) {
        constexpr int KEYS = decltype(keys)::value, GR = decltype(groups)::value;
        // item e's row is row0 + e NTHR / GR (a multiple of 8 apart, or the swizzle below would move)
        static_assert((NTHR / GR) % 8 == 0 && KEYS * GR == ITEMS * NTHR, "rows of a thread's items differ by whole swizzle groups");
        const int BP = min(p.P, KEYS);
        Places q;
#pragma unroll
        for (int e = 0; e < ITEMS; ++e) {
          const int key = (ct + e * NTHR) / GR, grp = (ct + e * NTHR) % GR + g0, in = key & (BP - 1);
          const uint32_t blk = (uint32_t)(key / BP) * L::v_code(BP);
          q.from[e] = blk + in * L::CODE + grp * 8;
          q.from_s[e] = blk + L::k_scale(BP) + in * L::SCALE + grp;
        }
        const int grp = ct % GR;
        q.row0 = ct / GR;
        // the halves of 8 lanes write different 16-byte columns: groups 4.. write their second chunk first
        q.flip = (grp >> 2) & 1;
        q.to = (grp >> 2) * (KEYS * 128) + q.row0 * 128 + ((((grp & 3) * 2 + q.flip) ^ (q.row0 & 7)) << 4);
        return q;
      };
      using std::integral_constant;
      constexpr int KK = TK / CG, VG = GP / CG, K_STEP = NTHR / GP, V_STEP = NTHR / VG;
      const Places pk = places(integral_constant<int, KK>{}, integral_constant<int, GP>{}, 0);
      const Places pv = CG == 1 ? pk : places(integral_constant<int, TK>{}, integral_constant<int, VG>{}, (int)rank * VG);
      int slot = 0;  // slots (and stages) so far: K and V of a tile in turn
      auto convert = [&](const Places& q, int step, int key0) {
        const int rs = slot % kRaw;
        if (!wait_warp(mbar::saddr(&raw_full[rs]), (slot / kRaw) & 1, &abort_flag)) return false;
        const uint32_t stage = s_rw + rs * C::RAW;
        uint2 w[ITEMS];
        uint32_t sc[ITEMS];
#pragma unroll
        for (int e = 0; e < ITEMS; ++e) {
          w[e] = lds_u64(stage + q.from[e]);
          sc[e] = lds_u8(stage + q.from_s[e]);
        }
        __syncwarp();
        if (lane == 0) mbar::arrive(mbar::saddr(&raw_empty[rs]));  // the stage is in registers
        if (!wait_warp(mbar::saddr(&kv_empty[slot % kSlots]), ((slot / kSlots) & 1) ^ 1, &abort_flag)) return false;
        const uint32_t out = s_kv + (slot % kSlots) * C::SLOT + q.to;
        if (key0 >= 0) {
          // V: slots that no row sees count as zero, and so does a NaN scale (put in at the end): 0 * NaN
#pragma unroll
          for (int e = 0; e < ITEMS; ++e) {
            if (key0 + q.row0 + e * step >= it.limit) sc[e] = 0;
            if ((sc[e] & 0x7F) == 0x7F) {
              store_all<CG>(mbar::saddr(const_cast<uint32_t*>(&nan_seen)), 1u);
              sc[e] = 0;
            }
          }
        }
#pragma unroll
        for (int e = 0; e < ITEMS; ++e) {
          const uint32_t s2 = __byte_perm(fp8x2_to_f16x2<CEK_E4M3>(sc[e]), 0, 0x1010);
          const uint32_t x = q.flip ? w[e].y : w[e].x, y = q.flip ? w[e].x : w[e].y;
          const uint32_t dst = out + e * step * 128;
          sts16(dst, hmul2(e2m1x2_to_f16x2<0>(x), s2), hmul2(e2m1x2_to_f16x2<1>(x), s2),
                hmul2(e2m1x2_to_f16x2<2>(x), s2), hmul2(e2m1x2_to_f16x2<3>(x), s2));
          sts16(dst ^ 16, hmul2(e2m1x2_to_f16x2<0>(y), s2), hmul2(e2m1x2_to_f16x2<1>(y), s2),
                hmul2(e2m1x2_to_f16x2<2>(y), s2), hmul2(e2m1x2_to_f16x2<3>(y), s2));
        }
        proxy_fence();
        __syncwarp();
        if (lane == 0) arrive_lead<CG>(mbar::saddr(&kv_full[slot % kSlots]));
        ++slot;
        return true;
      };
      for (int j = 0; j < n; ++j)
        if (!convert(pk, K_STEP, -1) || !convert(pv, V_STEP, (it.tile0 + j) * TK)) break;
    } else if (warp == 12) {
      // ---- matrix instructions, of a pair by its first CTA
      if (n > 0 && rank == 0) {
        bool ok = wait_warp(mbar::saddr(&q_full), 0, &abort_flag);
        auto qk = [&](int j, int st) {  // S = Q K^T into the stream's (tile's) buffer
          const uint32_t d = tmem + (NQ == 2 ? st : j & 1) * 128;
          const uint32_t a = s_q + st * (128 * D * 2), b = s_kv + ((2 * j) % kSlots) * C::SLOT;
          if (elect()) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              mma_ss<CG>(d, desc(a + (k >> 2) * (128 * 128) + (k & 3) * 32, 16), desc(b + (k >> 2) * (TK / CG * 128) + (k & 3) * 32, 16),
                     C::IDESC_QK, k > 0);
            commit<CG>(mbar::saddr(&s_full[NQ == 2 ? st : j & 1]));
          }
          __syncwarp();
        };
        auto pv = [&](int j, int st) {  // O += P V
          const uint32_t d = tmem + C::O_COL + st * D, a = tmem + (NQ == 2 ? st : j & 1) * 128;
          const uint32_t b = s_kv + ((2 * j + 1) % kSlots) * C::SLOT;
          if (elect()) {
#pragma unroll
            for (int k = 0; k < TK / 16; ++k)
              mma_ts<CG>(d, a + k * 8, desc(b + k * 2048, TK * 128), C::IDESC_PV, j > 0 || k > 0);
            commit<CG>(mbar::saddr(&o_done[st]));
          }
          __syncwarp();
        };
        auto release = [&](int i) {  // slot i once all products issued so far are done
          if (elect()) commit<CG>(mbar::saddr(&kv_empty[i % kSlots]));
          __syncwarp();
        };
        auto kv_ready = [&](int i) { return wait_warp(mbar::saddr(&kv_full[i % kSlots]), (i / kSlots) & 1, &abort_flag); };
        auto p_ready = [&](int j, int st) {
          const bool r = wait_warp(mbar::saddr(&p_full[NQ == 2 ? st : j & 1]), NQ == 2 ? j & 1 : (j >> 1) & 1, &abort_flag);
          fence_after();
          return r;
        };
        ok = ok && kv_ready(0);
        if (ok) {
          fence_after();
          for (int st = 0; st < NQ; ++st) qk(0, st);
          release(0);
        }
        for (int j = 0; j < n && ok; ++j) {
          if constexpr (NQ == 2) {
            for (int st = 0; st < 2 && ok; ++st) {
              ok = (st == 1 || kv_ready(2 * j + 1)) && p_ready(j, st);
              if (!ok) break;
              pv(j, st);
              if (st == 1) release(2 * j + 1);
              if (j + 1 < n) {
                if (st == 0) ok = kv_ready(2 * j + 2);
                if (!ok) break;
                fence_after();
                qk(j + 1, st);
                if (st == 1) release(2 * j + 2);
              }
            }
          } else {
            if (j + 1 < n) {
              ok = kv_ready(2 * j + 2);
              if (!ok) break;
              fence_after();
              qk(j + 1, 0);
              release(2 * j + 2);
            }
            ok = kv_ready(2 * j + 1) && p_ready(j, 0);
            if (!ok) break;
            pv(j, 0);
            release(2 * j + 1);
          }
        }
        if (elect()) commit<CG>(mbar::saddr(&drain));  // nothing of ours still runs when tensor memory is freed
        __syncwarp();
      }
      if (n > 0) wait(mbar::saddr(&drain), 0, &abort_flag);
    } else if (warp == 13) {
      // ---- pages
      int i = pages;
      for (; i < 2 * n; ++i) {
        if (!wait_warp(mbar::saddr(&raw_empty[i % kRaw]), ((i / kRaw) & 1) ^ 1, &abort_flag)) break;
        ask(i);
      }
      for (int a = i > kRaw ? i - kRaw : 0; a < i; ++a)  // no copy of ours is still landing
        wait(mbar::saddr(&raw_full[a % kRaw]), (a / kRaw) & 1, &abort_flag);
    }
  }

  sync_group<CG>();
  if (soft) {
    // ---- the row's output
    fence_after();
    uint32_t nan_groups = 0;
    if (nan_seen && real) {
      // rare: which groups of 16 channels see a value that is NaN
      const int k1 = min(hi, (it.tile0 + n) * TK);
      for (int key = max(lo, it.tile0 * TK); key < k1; ++key) {
        const int id = min(max(p.table[(int64_t)it.b * p.table_stride + key / p.P], 0), p.cache.num_pages - 1);
        const uint8_t* sca = p.cache.data + (int64_t)id * p.cache.page_stride + (int64_t)it.h * p.cache.head_stride +
                             L::v_scale(p.P) + (key % p.P) * L::SCALE;
        for (int gr = 0; gr < GP; ++gr) nan_groups |= (uint32_t)((sca[gr] & 0x7F) == 0x7F) << gr;
      }
    }
    const float inv = splits > 1 ? 1.f : l == 0.f ? 0.f : vf / l;
    float* part = p.partial + (int64_t)blockIdx.x * (ROWS * (D + 2));
    if (splits > 1 && real) {
      part[x * 128 + rr] = m == -INFINITY ? m : m * c;
      part[ROWS + x * 128 + rr] = l;
    }
    part += 2 * ROWS + (x * 128 + rr) * D;
#pragma unroll 1
    for (int i = 0; i < D; i += 32) {
      float o[32];
      if (n > 0) {
        tmem_ld32(tm_lane + C::O_COL + x * D + i, o);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int q = 0; q < 32; ++q) o[q] = 0.f;
      }
#pragma unroll
      for (int q = 0; q < 32; ++q) o[q] *= inv;
      if (nan_groups) {
#pragma unroll
        for (int q = 0; q < 32; ++q)
          if ((nan_groups >> ((i + q) >> 4)) & 1) o[q] = __int_as_float(0x7fffffff);
      }
      if (splits > 1 && real) {
#pragma unroll
        for (int q = 0; q < 32; q += 4) *reinterpret_cast<float4*>(part + i + q) = make_float4(o[q], o[q + 1], o[q + 2], o[q + 3]);
      } else {
        // by way of Q's place in shared memory: a row a thread would touch 32 lines a store
#pragma unroll
        for (int q = 0; q < 32; q += 8) {
          const int c16 = (i + q) / 8;
          sts16(s_q + x * (128 * D * 2) + (c16 >> 3) * (128 * 128) + rr * 128 + (((c16 & 7) ^ (rr & 7)) << 4),
                pack2<T>(o[q], o[q + 1]), pack2<T>(o[q + 2], o[q + 3]), pack2<T>(o[q + 4], o[q + 5]), pack2<T>(o[q + 6], o[q + 7]));
        }
      }
    }
    if (splits == 1) {
      __syncwarp();
      const int64_t to = real ? (int64_t)tok * p.ots + (int64_t)head * p.ohs : -1;
#pragma unroll 8
      for (int i = 0; i < 32; i += RPI) {
        const int r = i + lane / LPR, rw = (warp & 3) * 32 + r;
        const int64_t at = __shfl_sync(0xffffffffu, to, r);
        const uint4 u = mbar::lds16(s_q + x * (128 * D * 2) + (ch >> 3) * (128 * 128) + rw * 128 + (((ch & 7) ^ (rw & 7)) << 4));
        if (at >= 0) *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + at + ch * 8) = u;
      }
    }
    fence_before();
  }
  sync_group<CG>();
  fence_after();
  if (warp == 12) {
    if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// Joins the splits of a row: four warps a row, each every fourth split, then the
// four in order; D / 32 channels a lane.
template <typename T, int D, int NQ>
__global__ void __launch_bounds__(128)
attn_prefill_join_kernel(const AttnParams p, int row_blocks, int splits) {
  using C = Cfg<D, NQ, 1>;
  constexpr int ROWS = C::ROWS, E = D / 32, SIZE = ROWS * (D + 2);
  __shared__ float red[4][D], red_l[4];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const int b = blockIdx.z, h = blockIdx.y, row = blockIdx.x;
  const Request r = request_of<C::TK>(p, b);
  const int qi = row / p.group, tok = r.t0 + qi;
  if (row >= r.n * p.group || tok < 0 || tok >= p.tokens) return;
  const int rb = row / ROWS, col = row % ROWS;
  const int64_t item = ((int64_t)(row_blocks - 1 - rb) * p.requests + b) * p.cache.heads + h;
  const float* part = p.partial + item * splits * SIZE;
  float top = -INFINITY;
  for (int s = lane; s < splits; s += 32) top = fmaxf(top, part[(int64_t)s * SIZE + col]);
  top = warp_max(top);
  const float base = top == -INFINITY ? 0.f : top;
  float l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 8
  for (int s = sub; s < splits; s += 4) {
    const float* q = part + (int64_t)s * SIZE;
    const float w = ex2(q[col] - base);
    l += w * q[ROWS + col];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] += w * q[2 * ROWS + col * D + lane * E + e];
  }
#pragma unroll
  for (int e = 0; e < E; ++e) red[sub][lane * E + e] = o[e];
  if (lane == 0) red_l[sub] = l;
  __syncthreads();
  if (sub != 0) return;
  l = red_l[0] + red_l[1] + red_l[2] + red_l[3];
  const float inv = l == 0.f ? 0.f : p.cache.scales[p.cache.heads + h] / l;
  T* dst = static_cast<T*>(p.out) + (int64_t)tok * p.ots + (int64_t)(h * p.group + row - qi * p.group) * p.ohs + lane * E;
  uint32_t u[E / 2];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = (red[0][lane * E + e] + red[1][lane * E + e]) + (red[2][lane * E + e] + red[3][lane * E + e]);
#pragma unroll
  for (int e = 0; e < E / 2; ++e) u[e] = pack2<T>(o[2 * e] * inv, o[2 * e + 1] * inv);
  if constexpr (E == 2) *reinterpret_cast<uint32_t*>(dst) = u[0];
  else if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(u[0], u[1]);
  else *reinterpret_cast<uint4*>(dst) = make_uint4(u[0], u[1], u[2], u[3]);
}

struct Plan {
  int nq, cg, row_blocks, splits;
  int64_t items, partial_bytes;
};
inline Plan plan_of(int64_t d, int64_t requests, int64_t tokens, int64_t heads, int64_t group, int64_t max_q, int64_t max_seq) {
  Plan r;
  const int64_t rows = max_q * group;
  r.nq = d == 256 || rows <= 128 ? 1 : 2;
  // row blocks of all requests together: if each were as long as the longest, and at most by
  // the number of tokens
  auto count = [&](int64_t block, bool* packed) {
    r.row_blocks = (int)((rows + block - 1) / block);
    const int64_t loose = requests * r.row_blocks, tight = tokens * group / block + requests;
    *packed = loose > 2 * tight;
    if (*packed) r.row_blocks = 0;
    return heads * (*packed ? tight : loose);
  };
  bool packed;
  r.cg = r.splits = 1;
  r.items = count(128 * r.nq, &packed);
  // too few row blocks for the SMs: split their keys, at least four tiles of the longest bound a
  // piece (behind a window most pieces have none: their blocks write an empty piece)
  const int64_t tiles = (max_seq + (d == 256 ? 63 : 127)) / (d == 256 ? 64 : 128);
  if (!packed && r.items < cek_host::sm_count() && tiles >= 8)
    r.splits = (int)std::max<int64_t>(1, std::min<int64_t>(cek_host::sm_count() / r.items, tiles / 4));
  r.partial_bytes = r.splits > 1 ? r.items * r.splits * 128 * r.nq * (d + 2) * (int64_t)sizeof(float) : 0;
  // enough work for all SMs in pairs: 1115 us instead of 1154 (8192 tokens, 64/8 heads of 128)
  if ((d == 256 || (d == 128 && r.nq == 2)) && r.splits == 1 && r.items >= 2 * cek_host::sm_count()) {
    r.cg = 2;
    r.items = count(256 * r.nq, &packed);
  }
  return r;
}

template <typename T, int D, int NQ, int CG>
int launch(const AttnParams& p, const Plan& r, cudaStream_t st) {
  using C = Cfg<D, NQ, CG>;
  static cek_host::DeviceSlots attr;
  if (!cek_host::ensure_smem_attr(attr, attn_prefill_kernel<T, D, NQ, CG>, C::SMEM)) return CEK_ERR_LAUNCH;
  const int64_t blocks = r.items * r.splits * CG;
  if (blocks > INT32_MAX) return CEK_ERR_INVALID_ARG;
  if constexpr (CG == 2) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute a[2];
    a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a[0].val.programmaticStreamSerializationAllowed = cek_host::pdl_enabled() ? 1 : 0;
    a[1].id = cudaLaunchAttributeClusterDimension;
    a[1].val.clusterDim.x = 2;
    a[1].val.clusterDim.y = a[1].val.clusterDim.z = 1;
    cfg.attrs = a;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, attn_prefill_kernel<T, D, NQ, CG>, p, r.row_blocks, r.splits) == cudaSuccess ? CEK_OK
                                                                                                              : CEK_ERR_LAUNCH;
  } else {
    int s = cek_host::launch_pdl(attn_prefill_kernel<T, D, NQ, CG>, dim3((unsigned)blocks), dim3(kThreads), C::SMEM, st, p,
                                 r.row_blocks, r.splits);
    if (s != CEK_OK || r.splits == 1) return s;
    const dim3 grid((unsigned)(p.max_q * p.group), (unsigned)p.cache.heads, (unsigned)p.requests);
    return cek_host::launch_pdl(attn_prefill_join_kernel<T, D, NQ>, grid, dim3(128), 0, st, p, r.row_blocks, r.splits);
  }
}
template <typename T>
int launch_t(int64_t d, const AttnParams& p, const Plan& r, cudaStream_t st) {
  if (d == 64) return r.nq == 1 ? launch<T, 64, 1, 1>(p, r, st) : launch<T, 64, 2, 1>(p, r, st);
  if (d == 256) return r.cg == 1 ? launch<T, 256, 1, 1>(p, r, st) : launch<T, 256, 1, 2>(p, r, st);
  if (r.nq == 1) return launch<T, 128, 1, 1>(p, r, st);
  return r.cg == 1 ? launch<T, 128, 2, 1>(p, r, st) : launch<T, 128, 2, 2>(p, r, st);
}
}  // namespace pf

int64_t prefill_workspace(int64_t d, int64_t requests, int64_t tokens, int64_t heads, int64_t group, int64_t max_q,
                          int64_t max_seq) {
  return pf::plan_of(d, requests, tokens, heads, group, max_q, max_seq).partial_bytes;
}
int prefill_launch(int dtype, int64_t d, const AttnParams& p, int64_t max_seq, cudaStream_t st) {
  const pf::Plan r = pf::plan_of(d, p.requests, p.tokens, p.cache.heads, p.group, p.max_q, max_seq);
  return dtype == CEK_F16 ? pf::launch_t<__half>(d, p, r, st) : pf::launch_t<__nv_bfloat16>(d, p, r, st);
}
bool prefill_timeouts(unsigned long long* v) {
  return cudaMemcpyFromSymbol(v, g_timeouts_prefill, sizeof(*v)) == cudaSuccess;
}
}  // namespace kv4
}  // namespace cek

