// Causal attention over packed prompts on the 5th-generation tensor cores
// (sm_100a): grouped heads, sequences of different lengths one after another,
// keys that may begin before the queries (a prompt chunk behind its history).
//
//   out[i, h] = softmax_k(q[i, h] . k[k, h / G] * scale) v[k, h / G]
//   over the keys k <= i + (keys - queries) of i's sequence
//
// Two matrix products of 4 * 128 flops per visible pair bound it, so the tensor
// core must never wait for long: an SM works on two tiles of 128 queries that take
// turns, and while one tile's scores are in softmax the other's products run. The
// two are one CTA's (256 queries of one (sequence, head), long prompts) or two
// CTAs' (short ones). Warps of a CTA:
//   4 per tile      softmax, one thread per query row: S (128 keys) goes
//                   TMEM -> registers in chunks, P goes back in 16 bits over S's
//                   own columns, in two halves of 64 keys, so that the first half
//                   is multiplied while the second is still in softmax. P never
//                   touches shared memory.
//   next            TMA: Q, then K and V blocks of 128 keys through a ring
//   last            MMA issue, per block and tile: O += P V for both halves, then the
//                   next S = Q K^T over the columns that P leaves. Products of
//                   one warp run in order, so no barrier says that.
// TMEM: S, 128 fp32 columns a tile, then O, 128 a tile.
//
// 16384 tokens, 32 + 8 heads: 1.99 to 2.06 ms on different GPUs, 1.07 to 1.10 PFLOP/s. Of the 3500 cycles of a block
// of both tiles products take 2050, and at 1 kW the SM clock is at 1.55 GHz, so what
// shortens the cycles without saving energy gains nothing. Measured and not kept:
//   P by polynomial on the FMA pipe for a quarter of the keys, scores prefetched
//   across P's halves: 3380 cycles at 1.52 GHz, 2.00 ms
//   an issuing warp for each tile of a CTA: the tiles fall into step, 2.30 ms
//   steps of 64 keys with two S buffers per tile: 2.16 ms, since a 128 x 64 product
//   reads 6 KB of shared memory in 32 cycles' work
//
// P = 2^(s - m) needs no exact maximum, only one reference m for P, the row sum and
// O that keeps P within 16 bits: m is the row's maximum over its first block (that
// has a score above -inf) and moves only when the sum of 64 P exceeds 2^8 (so no P does otherwise). Then the
// half is looked at again, O and the sum are rescaled (a read and write of 128
// columns) and its P recomputed: rare after the first block, and until then no
// maximum is taken at all. Sums and maxima are fp32;
// P is rounded to the 16-bit type of V, its only rounding.
//
// A masked key's P is 0, but 0 * NaN is not: in the blocks that need a mask (the
// diagonal and a sequence's end) the V rows behind the end are cleared in shared
// memory, and so is a single value that is not finite. The first key with +inf, -inf
// and NaN is kept for each channel, and the queries that see it get it added to
// that channel of their output, as the product does in a block without a mask.
#include <cuda_runtime.h>

#include <type_traits>

#include "ps_common.cuh"
#include "ps_host.h"

namespace ps {
namespace pra {

constexpr int kD = 128;
constexpr int kTile = 128;              // queries of a tile, keys of a block
constexpr int kTileBytes = kTile * kD * 2;
constexpr int kHalf = kTileBytes / 2;   // one 64-column TMA box (128 rows x 128 bytes)
constexpr int kKeys = 64;               // keys of half a block
constexpr int kBadBytes = 3 * kD * 4;   // first key with +inf, -inf, NaN in each channel
constexpr int kNoKey = 0x7fffffff;
// What a CTA is made of: kTiles tiles of queries.
template <int kTiles>
struct Shape {
  static constexpr int kRows = kTile * kTiles;           // queries
  static constexpr int kSlots = kTiles == 2 ? 5 : 2;     // of the K / V ring
  static constexpr int kThreads = (kTiles * 4 + 2) * 32;
  static constexpr int kCtas = 3 - kTiles;               // resident on an SM
  static constexpr int kSmem = 1024 + kTileBytes * (kTiles + kSlots) + 256 + kBadBytes;
  static constexpr int kTmemCols = 256 * kTiles;
  static constexpr int kTmemO = 128 * kTiles;            // S tiles from 0, O tiles from here
};
constexpr float kMaxSum = 256.f;        // of 64 P, before the reference moves

struct Args {
  void* out;
  long long o_stride;
  const int32_t* cu_q;  // [n + 1]
  const int32_t* cu_k;
  int n, Tq, Tk, n_heads, group, bf16;
  int wide;  // out's rows are 32-byte aligned
  float scale_log2;
  int32_t* status;
};

// A value that all lanes share, known as such to the compiler (a warp reduction
// ends in a uniform register): loops over it and addresses made from it stay in
// the uniform data path, which the product instructions take their operands from.
PS_DEV uint32_t uniform(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

// The MMA warp runs as one: every lane computes the same operands and waits on
// the same barriers, and the instructions themselves are predicated to one lane.
// Inside a single-lane branch each operand would have to be moved to a uniform
// register first, which made issuing a product take longer than the product
// (155 instead of 64 cycles).
// D[tmem] (+)= A[smem desc] * B[smem desc], kind::f16.
PS_DEV void mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                   uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The same with A[tmem, 16-bit pairs].
PS_DEV void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                   uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
PS_DEV void mma_commit(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(
          bar)
      : "memory");
}
PS_DEV bool try_wait_at(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// mbar_wait on a shared-memory address.
PS_DEV bool wait_at(uint32_t bar, uint32_t parity, int32_t* status) {
  if (try_wait_at(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    for (int i = 0; i < 64; ++i)
      if (try_wait_at(bar, parity)) return true;
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      set_status(status, PS_ERR_TIMEOUT);
      return false;
    }
  }
}

#define PS_R32(r)                                                                             \
  "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),         \
      "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), \
      "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),           \
      "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),           \
      "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
#define PS_RW16(r)                                                                            \
  "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),         \
      "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), \
      "+r"(r[14]), "+r"(r[15])
#define PS_IN32(r)                                                                            \
  "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),     \
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),       \
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),     \
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),     \
      "r"(r[29]), "r"(r[30]), "r"(r[31])

// 32 columns of this thread's lane; complete after ld_wait on the same registers.
PS_DEV void ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : PS_R32(r)
      : "r"(taddr));
}
PS_DEV void ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Ties registers to the wait above: no use of them moves in front of it.
PS_DEV void after_wait(uint32_t* r) {
  asm volatile("" : PS_RW16(r)::"memory");
  asm volatile("" : PS_RW16((r + 16))::"memory");
}
PS_DEV void st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31};" ::PS_IN32(r),
      "r"(taddr)
      : "memory");
}

PS_DEV float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
PS_DEV uint32_t pack16(float lo, float hi);
template <>
PS_DEV uint32_t pack16<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
PS_DEV uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The row's largest score of kCols columns (raw, before the scale).
template <int kCols>
PS_DEV float row_max(uint32_t s_addr, bool masked, int lim) {
  float mx = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < kCols; c += 32) {
    uint32_t s[32];
    ld32(s_addr + c, s);
    ld_wait();
    after_wait(s);
#pragma unroll
    for (int i = 0; i < 32; ++i)
      mx = fmaxf(mx, masked && c + i >= lim ? -INFINITY : __uint_as_float(s[i]));
  }
  return mx;
}

// P = 2^(s * scale + neg) of half a block, the row's 64 scores, in 16 bits, and
// their sum. P stays in registers until the caller knows that neg was good
// enough; S is then overwritten.
template <typename T>
PS_DEV float softmax_half(uint32_t s_addr, bool masked, int lim, float scale, float neg,
                          uint32_t* p) {
  const uint64_t scale2 = f32x2(scale, scale), neg2 = f32x2(neg, neg);
  uint64_t l0 = f32x2(0.f, 0.f), l1 = l0;
  uint32_t s[2][32];
  ld32(s_addr, s[0]);
#pragma unroll
  for (int c = 0; c < kKeys / 32; ++c) {
    uint32_t* v = s[c & 1];
    ld_wait();
    after_wait(v);
    if (c + 1 < kKeys / 32) ld32(s_addr + 32 * (c + 1), s[(c + 1) & 1]);
    if (masked) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (32 * c + i >= lim) v[i] = 0xff800000u;  // -inf
    }
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      float x0, x1, y0, y1;
      f32x2_split(f32x2_fma(f32x2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), scale2, neg2), x0, x1);
      f32x2_split(f32x2_fma(f32x2(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])), scale2, neg2), y0,
             y1);
      x0 = exp2_ftz(x0);
      x1 = exp2_ftz(x1);
      y0 = exp2_ftz(y0);
      y1 = exp2_ftz(y1);
      l0 = f32x2_add(l0, f32x2(x0, x1));
      l1 = f32x2_add(l1, f32x2(y0, y1));
      p[16 * c + i / 2] = pack16<T>(x0, x1);
      p[16 * c + i / 2 + 1] = pack16<T>(y0, y1);
    }
  }
  float s0, s1;
  f32x2_split(f32x2_add(l0, l1), s0, s1);
  return s0 + s1;
}

// Whether 8 16-bit values are all finite (an exponent of ones is not).
template <typename T>
PS_DEV bool finite8(const uint4& u) {
  const uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  bool fin = true;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    fin = fin && (w[i] & e) != e && ((w[i] >> 16) & e) != e;
  return fin;
}

// Clear the values of one row's 64 channels (128 swizzled bytes of key `key`) that are not
// finite, noting their keys by kind and channel. Rare, so small rather than fast.
template <typename T>
PS_DEV void clear_bad(uint8_t* row, int key, int ch0, int* bad) {
#pragma unroll 1
  for (int c = 0; c < 64; ++c) {
    T* p = reinterpret_cast<T*>(row + ((((c >> 3) ^ key) & 7) << 4)) + (c & 7);
    const float x = to_f32<T>(*p);
    if (fabsf(x) <= 3.402823466e38f) continue;
    const int kind = x != x ? 2 : (x > 0.f ? 0 : 1);
    atomicMin(bad + kind * kD + ch0 + c, key);
    __threadfence_block();  // whoever finds it cleared finds its key
    *p = from_f32<T>(0.f);
  }
}

// With R queries to a CTA, sequence i owns slots [cu_q[i] / R + i, cu_q[i + 1] / R + i + 1): at
// least as many as it has tiles, found by a search, no scan of lengths (every lane of a warp
// calls it).
struct Item {
  int q0, k0, lq, lk, row;  // first rows, lengths, first query of this CTA
  bool live;
};

PS_DEV Item item_at(const Args& a, int slot, int kRows) {
  const int lane = threadIdx.x & 31;
  int lo = 0, count = a.n;  // the last i of [lo, lo + count) whose slots begin by `slot`
  while (count > 1) {       // 32 of them looked at together: the loads are what takes time
    const int step = (count + 31) / 32, i = lo + lane * step;
    const bool le = lane == 0 || (lane * step < count && a.cu_q[i] / kRows + i <= slot);
    const int last = 31 - __clz((int)__ballot_sync(0xffffffffu, le));
    lo += last * step;
    count = min(step, count - last * step);
  }
  Item it;
  it.q0 = a.cu_q[lo];
  it.k0 = a.cu_k[lo];
  const int q1 = a.cu_q[lo + 1], k1 = a.cu_k[lo + 1];
  const bool ok = it.q0 >= 0 && q1 >= it.q0 && q1 <= a.Tq && it.k0 >= 0 && k1 >= it.k0 && k1 <= a.Tk;
  it.lq = ok ? q1 - it.q0 : 0;
  it.lk = ok ? k1 - it.k0 : 0;
  const int tiles = (it.lq + kRows - 1) / kRows;
  const int t = slot - (it.q0 / kRows + lo);
  it.live = ok && t >= 0 && t < tiles;
  it.row = (tiles - 1 - t) * kRows;  // most work first
  if (!ok && threadIdx.x == 0) set_status(a.status, PS_ERR_BAD_INDEX);
  return it;
}

// Key blocks that tile t (rows row .. of lq) sees.
PS_DEV int blocks_of(const Item& it, int t) {
  const int first = it.row + t * kTile;
  if (first >= it.lq) return 0;
  const int last = min(it.lq, first + kTile) - 1;
  const int keys = last + 1 + it.lk - it.lq;  // visible to the last row
  return keys > 0 ? (keys + kTile - 1) / kTile : 0;
}

template <typename T, int kTiles>
__global__ void __launch_bounds__(Shape<kTiles>::kThreads, Shape<kTiles>::kCtas)
    prompt_attention_kernel(const __grid_constant__ CUtensorMap tq,
                            const __grid_constant__ CUtensorMap tk,
                            const __grid_constant__ CUtensorMap tv, const Args a) {
  constexpr int kSlots = Shape<kTiles>::kSlots, kTmemO = Shape<kTiles>::kTmemO;
  constexpr int kTma = 4 * kTiles, kMma = kTma + 1;  // warps
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t pad = (1024 - (smem_u32(smem_raw) & 1023)) & 1023;
  uint8_t* sQ = smem_raw + pad;             // [2] tiles
  uint8_t* sKV = sQ + kTiles * kTileBytes;  // ring: K0 V0 K1 V1 ...
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + kSlots * kTileBytes);
  uint64_t* q_full = bars;             // [2]
  uint64_t* kv_full = q_full + 2;      // [kSlots]
  uint64_t* kv_empty = kv_full + kSlots;
  uint64_t* s_full = kv_empty + kSlots;  // [2]
  uint64_t* p_full = s_full + 2;         // [2 tiles][2 halves]
  uint64_t* pv_done = p_full + 4;        // [2]: O += P V of a block's first half
  uint64_t* o_done = pv_done + 2;        // [2]
  uint64_t* drain = o_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* poison = reinterpret_cast<int*>(tmem_slot + 2);  // first key with a value cleared
  int* bad = reinterpret_cast<int*>(bars + 32);         // [3 kinds][128 channels]: the same of each

  const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const bool producer = warp == kTma && lane == 0;
  if (warp == kMma) {
    tmem_alloc(tmem_slot, Shape<kTiles>::kTmemCols);
    tmem_relinquish();
  }
  if (producer) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(pv_done + i, 1);
      mbar_init(o_done + i, 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(p_full + i, 4);
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 1);
    }
    mbar_init(drain, 1);
    abort_flag[0] = 0;
    poison[0] = kNoKey;
    fence_mbar_init();
  }
  for (int i = threadIdx.x; i < 3 * kD; i += Shape<kTiles>::kThreads) bad[i] = kNoKey;
  __syncwarp();
  pdl_wait();

  const int h = blockIdx.x % a.n_heads;
  const Item it = item_at(a, blockIdx.x / a.n_heads, Shape<kTiles>::kRows);
  const int nb0 = (int)uniform(it.live ? blocks_of(it, 0) : 0);
  const int nb1 = (int)uniform(it.live && kTiles > 1 ? blocks_of(it, 1) : 0);
  const int nb = max(nb0, nb1);

  // Key or value block of ring item i: K0 V0 K1 V1 ...
  const uint64_t pol = l2_policy_evict_last();  // a head's K / V serve all its tiles
  auto load_kv = [&](int i) {
    const int st = i % kSlots, c = (h / a.group) * kD;
    const CUtensorMap* tm = i & 1 ? &tv : &tk;
    const int r = it.k0 + (i >> 1) * kTile;
    uint8_t* dst = sKV + st * kTileBytes;
    mbar_arrive_expect_tx(kv_full + st, kTileBytes);
    tma_load_2d(dst, tm, kv_full + st, c, r, pol);
    tma_load_2d(dst + kHalf, tm, kv_full + st, c + 64, r, pol);
  };
  // What the first products need is on its way before the warps meet and TMEM is known
  if (producer && nb > 0) {
    load_kv(0);
    for (int t = 0; t < kTiles; ++t) {
      if ((t ? nb1 : nb0) == 0) continue;
      mbar_arrive_expect_tx(q_full + t, kTileBytes);
      const int r = it.q0 + it.row + t * kTile;
      tma_load_2d(sQ + t * kTileBytes, &tq, q_full + t, h * kD, r, pol);
      tma_load_2d(sQ + t * kTileBytes + kHalf, &tq, q_full + t, h * kD + 64, r, pol);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  // Not before every CTA has its TMEM: the next kernel's CTAs allocate theirs before they
  // wait for this grid.
  pdl_launch_dependents();

  if (warp >= kTma) {
    // ------------------------------------------------------------- producer
    if (producer && nb > 0) {
      int i = 1;
      for (; i < 2 * nb; ++i) {
        if (abort_flag[0] ||
            !mbar_wait(kv_empty + i % kSlots, ((i / kSlots) & 1) ^ 1, a.status)) {
          abort_flag[0] = 1;
          break;
        }
        load_kv(i);
      }
      if (abort_flag[0]) {  // let every issued copy land before the CTA exits
        if (nb0) mbar_wait(q_full, 0, a.status);
        if (nb1) mbar_wait(q_full + 1, 0, a.status);
        for (int n = max(0, i - kSlots); n < i; ++n)
          mbar_wait(kv_full + n % kSlots, (n / kSlots) & 1, a.status);
      }
    }
    // ------------------------------------------------------------------ MMA
    if (warp == kMma && nb > 0) {
      const uint32_t idesc_s = idesc_f16(a.bf16, 0, 0, kTile, kTile);  // Q, K both K-major
      const uint32_t idesc_o = idesc_f16(a.bf16, 0, 1, kTile, kD);     // P K-major, V MN-major
      const uint64_t q_desc = smem_desc_sw128(smem_u32(sQ), 16, 1024);
      const uint64_t k_desc = smem_desc_sw128(smem_u32(sKV), 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(smem_u32(sKV), kHalf, 1024);
      // Between a wait and the next product the queue of issued products covers
      // about 100 cycles, so this loop keeps addresses, slots and phases in
      // registers and waits as rarely as it can: once for each P, once for
      // each K and V block. What a wait that ran out leads to is decided once
      // a block; an aborting warp is not looked for, its waits run out too.
      const uint32_t bar0 = smem_u32(bars);
      const uint32_t kv_full_a = bar0 + 16, kv_empty_a = kv_full_a + 8 * kSlots;
      const uint32_t s_full_a = kv_empty_a + 8 * kSlots, p_full_a = s_full_a + 16;
      const uint32_t pv_done_a = p_full_a + 32, o_done_a = pv_done_a + 16;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        ok = wait_at(bar, parity, a.status) && ok;
      };
      // S_t = Q_t K^T, K's block in ring slot `slot`
      auto scores = [&](int t, int slot) {
        const uint64_t qd = q_desc + (t * kTileBytes >> 4);
        const uint64_t kd = k_desc + (uint32_t)(slot * (kTileBytes >> 4));
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk) {
          const uint64_t o = ((kk >> 2) * kHalf + (kk & 3) * 32) >> 4;
          mma_ss(tmem + t * kTile, qd + o, kd + o, idesc_s, kk > 0 ? 1u : 0u);
        }
        mma_commit(s_full_a + 8 * t);
      };
      // O_t += P_t V of one half of a block
      auto values = [&](int t, int half, int slot, bool first) {
        const uint64_t vd = v_desc + (uint32_t)(slot * (kTileBytes >> 4) + half * (kKeys * 128 >> 4));
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          mma_ts(tmem + kTmemO + t * kD, tmem + t * kTile + half * kKeys + kk * 8,
                 vd + (kk * 2048 >> 4), idesc_o, kk > 0 || !first ? 1u : 0u);
      };
      wait(kv_full_a, 0);
      if (nb0) wait(bar0, 0);
      if (nb1) wait(bar0 + 8, 0);
      tc_fence_after();
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        if (nb0) scores(0, 0);
        if (nb1) scores(1, 0);
        mma_commit(kv_empty_a);
      }
      // block j: V in slot vs, and the next block's K in slot ks
      int vs = 1, ks = 2 % kSlots;
      uint32_t vph = 0, kph = 2 / kSlots;
#pragma unroll 1
      for (int j = 0; ok && j < nb; ++j) {
        wait(kv_full_a + 8 * vs, vph);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const int n = t ? nb1 : nb0;
          if (j < n) {
            wait(p_full_a + 16 * t, j & 1);
            tc_fence_after();
            values(t, 0, vs, j == 0);
            mma_commit(pv_done_a + 8 * t);
            // The next block's K is waited for where P's second half is not there yet
            // (at the loop's top it delayed P V: 8 heads of 4096 tokens 66 and 62 us)
            if (j + 1 < nb && t == (j < nb0 ? 0 : 1)) wait(kv_full_a + 8 * ks, kph);
            wait(p_full_a + 16 * t + 8, j & 1);
            tc_fence_after();
            values(t, 1, vs, false);
            if (j + 1 < n)
              scores(t, ks);
            else
              mma_commit(o_done_a + 8 * t);
          }
        }
        // Everything that reads these slots has been issued: free them when done
        mma_commit(kv_empty_a + 8 * vs);
        if (j + 1 < nb) mma_commit(kv_empty_a + 8 * ks);
        vs += 2, ks += 2;
        if (vs >= kSlots) vs -= kSlots, vph ^= 1;
        if (ks >= kSlots) ks -= kSlots, kph ^= 1;
        ok = __all_sync(0xffffffffu, ok);
      }
      if (!ok) abort_flag[0] = 1;
      // every MMA of this CTA completes before TMEM is released
      mma_commit(smem_u32(drain));
      mbar_wait(drain, 0, a.status);
    }
  } else {
    // -------------------------------------------------------------- softmax
    const int t = kTiles > 1 ? warp >> 2 : 0;
    const int r = (warp & 3) * 32 + lane;  // TMEM lane = row of the tile
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_addr = tmem + kTmemO + t * kD + lane_off;
    const int first = it.row + t * kTile;
    const int row = first + r;
    const int my_nb = t ? nb1 : nb0;
    const int seen = row + 1 + it.lk - it.lq;  // keys this row sees: [0, seen)
    const int all_seen = first + 1 + it.lk - it.lq;  // seen by every row of the tile
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    const uint32_t s_addr = tmem + t * kTile + lane_off;
    for (int j = 0; j < my_nb && ok; ++j) {
      const bool got = !abort_flag[0] && wait_at(smem_u32(s_full + t), j & 1, a.status);
      if (!__all_sync(0xffffffffu, got)) {  // the warp leaves together (collective TMEM ops)
        ok = false;
        break;
      }
      tc_fence_after();
      const bool masked = j * kTile + kTile > all_seen;  // the diagonal, or the end
      const int lim = seen - j * kTile;                  // this row's keys of the block
      // Rows with nothing to go by yet take their maximum: all of them in the first block, and
      // later those whose every score so far was -inf (their P, sum and O are still 0).
      if (__any_sync(0xffffffffu, m == -INFINITY)) {
        const float mx = row_max<kTile>(s_addr, masked, lim) * a.scale_log2;
        if (m == -INFINITY) m = mx;
      }
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        const uint32_t h_addr = s_addr + half * kKeys;
        const int hlim = lim - half * kKeys;
        uint32_t p[32];
        const float neg = m == -INFINITY ? 0.f : -m;
        float lsum = softmax_half<T>(h_addr, masked, hlim, a.scale_log2, neg, p);
        if (__any_sync(0xffffffffu, lsum > kMaxSum)) {
          // tcgen05 loads and stores are warp-collective: rows that stay scale by 1
          const float mx = row_max<kKeys>(h_addr, masked, hlim) * a.scale_log2;
          const bool moved = lsum > kMaxSum && mx > m;
          const float alpha = moved ? exp2_ftz(m - mx) : 1.f;
          if (moved) m = mx;
          l *= alpha;
          // O is at rest: S(j) says that block j - 1 is in it, and of this block
          // only the first half can be on its way, when this is the second.
          bool rest = true;
          if (half) rest = mbar_wait(pv_done + t, j & 1, a.status);
          if (!__all_sync(0xffffffffu, rest)) {
            ok = false;
            break;
          }
          if (j > 0 || half) {
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < kD; c += 32) {
              uint32_t o[32];
              ld32(o_addr + c, o);
              ld_wait();
              after_wait(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              st32(o_addr + c, o);
            }
          }
          lsum = softmax_half<T>(h_addr, masked, hlim, a.scale_log2, moved ? -mx : neg, p);
        }
        st32(h_addr, p);
        l += lsum;
        if (masked) {
          // V landed? (it follows K in the ring). Two threads to a row, 128 bytes each.
          const int i = 2 * j + 1, key = j * kTile + half * kKeys + (r & (kKeys - 1));
          if (mbar_wait(kv_full + i % kSlots, (i / kSlots) & 1, a.status)) {
            uint8_t* v = sKV + (i % kSlots) * kTileBytes + (r >> 6) * kHalf +
                         (key & (kTile - 1)) * 128;
            if (key < it.lk) {
              bool fin = true;
#pragma unroll
              for (int c = 0; c < 8; ++c)  // 16-byte chunks, rotated by row: no bank conflicts
                fin &= finite8<T>(*reinterpret_cast<const uint4*>(v + (((c + r) & 7) << 4)));
              if (!fin) {
                atomicMin(poison, key);
                clear_bad<T>(v, key, (r >> 6) * 64, bad);
              }
            } else {
#pragma unroll
              for (int c = 0; c < 8; ++c)
                *reinterpret_cast<uint4*>(v + (((c + r) & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          fence_proxy_async_smem();  // the cleared rows -> the tensor core's view
        }
        __syncwarp();
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 2 * t + half);
      }
    }
    const bool live = it.live && row < it.lq;
    bool fin = ok;
    if (my_nb > 0) fin = ok && !abort_flag[0] && mbar_wait(o_done + t, 0, a.status);
    fin = __all_sync(0xffffffffu, fin);
    if (!fin) abort_flag[0] = 1;
    if (fin && it.live) {
      tc_fence_after();
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // a row that sees no key: 0
      T* orow = reinterpret_cast<T*>(a.out) + (size_t)(it.q0 + row) * a.o_stride + h * kD;
#pragma unroll 1
      for (int c = 0; c < kD; c += 32) {
        uint32_t o[32];
        if (my_nb > 0) {
          ld32(o_addr + c, o);
          ld_wait();
          after_wait(o);
        }
        if (live) {
#pragma unroll
          for (int i = 0; i < 32; i += 16) {
            uint32_t w[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
            if (my_nb > 0 && inv != 0.f) {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                w[k] = pack16<T>(__uint_as_float(o[i + 2 * k]) * inv,
                                 __uint_as_float(o[i + 2 * k + 1]) * inv);
            }
            // a warp's 32 rows are 32 sectors of different lines; with 16-byte stores each is
            // touched twice (8 prompts of 512 to 1024 tokens: 87 and 82 us; one of 16384:
            // 2.00 and 1.99 ms)
            if (a.wide) {
              st_32bytes(orow + c + i, w);
            } else {
              reinterpret_cast<uint4*>(orow + c + i)[0] = make_uint4(w[0], w[1], w[2], w[3]);
              reinterpret_cast<uint4*>(orow + c + i)[1] = make_uint4(w[4], w[5], w[6], w[7]);
            }
          }
        }
      }
      if (live && seen > *reinterpret_cast<volatile int*>(poison)) {
        const volatile int* key = bad;
#pragma unroll 1
        for (int c = 0; c < kD; ++c) {
          float x = 0.f;
          if (seen > key[c]) x += __uint_as_float(0x7f800000u);
          if (seen > key[kD + c]) x -= __uint_as_float(0x7f800000u);
          if (seen > key[2 * kD + c]) x = __uint_as_float(0x7fc00000u);
          if (x != 0.f) orow[c] = from_f32<T>(to_f32<T>(orow[c]) + x);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc(tmem, Shape<kTiles>::kTmemCols);
  }
}

}  // namespace pra
}  // namespace ps

using namespace ps;

extern "C" int ps_prompt_attention(const void* q, long long q_stride, const void* k,
                                   long long k_stride, const void* v, long long v_stride,
                                   void* out, long long o_stride, const int32_t* cu_q,
                                   const int32_t* cu_k, int n_seqs, int Tq, int Tk, int n_heads,
                                   int n_kv_heads, float scale, int dtype, int32_t* status,
                                   ps_stream_t stream) {
  PS_CHECK_ARG(n_seqs >= 0 && Tq >= 0 && Tk >= 0 && n_heads > 0 && n_kv_heads > 0 &&
               n_heads % n_kv_heads == 0);
  PS_CHECK_ARG(dtype == PS_DTYPE_F16 || dtype == PS_DTYPE_BF16);
  PS_CHECK_ARG(scale > 0.f && scale < kMaxScale);
  if (n_seqs == 0 || Tq == 0) return PS_OK;
  PS_CHECK_ARG(q && out && cu_q && cu_k && aligned16(q) && aligned16(out));
  PS_CHECK_ARG(Tk == 0 || (k && v && aligned16(k) && aligned16(v)));
  PS_CHECK_ARG(q_stride >= (long long)n_heads * pra::kD && q_stride % 8 == 0 &&
               o_stride >= (long long)n_heads * pra::kD && o_stride % 8 == 0);
  PS_CHECK_ARG(Tk == 0 || (k_stride >= (long long)n_kv_heads * pra::kD && k_stride % 8 == 0 &&
                           v_stride >= (long long)n_kv_heads * pra::kD && v_stride % 8 == 0));
  // By the mean length, which is what the host knows: two CTAs of one tile on an SM
  // (128 queries each) waste less of a short sequence and hide each other's start
  // (64 prompts of 64 to 128 tokens, 32 + 8 heads: 65 us, one CTA of two tiles 118; 8 of
  // 512 to 1024: 81 and 101); two tiles read each K and V block once for twice the
  // queries, which wins behind some 4096 (one prompt of 4096: 138 and 140 us, of 8192:
  // 547 and 515, of 16384: 2084 and 1976; with 32 + 32 heads of 4096: 158 and 172, of
  // 8192: 524 and 508, of 16384: 2157 and 1948). The rule looks at keys alone: with few
  // queries behind them one tile stays ahead by 1 to 6% (256 queries behind 8192 keys: 130 and
  // 138 us, behind 16384: 245 and 255, behind 65536: 915 and 946), and a long prompt among
  // many short ones gets one (one of 16384 and 31 of 64: 2082 and 2014).
  const bool one = Tk <= 4096ll * n_seqs;
  const int rows = pra::kTile * (one ? 1 : 2);
  const long long grid = ((long long)Tq / rows + n_seqs) * n_heads;
  if (grid > 0x7fffffffll || Tk > (1 << 30) || Tq > (1 << 30)) return PS_ERR_UNSUPPORTED;
  const int device = current_device();
  if (!is_sm100(device)) return PS_ERR_UNSUPPORTED;
  const bool bf = dtype == PS_DTYPE_BF16;
  const uint32_t box[2] = {64, (uint32_t)pra::kTile};
  CUtensorMap tq, tk, tv;
  auto make = [&](CUtensorMap* map, const void* p, long long stride, int heads, int rows) {
    const uint64_t dims[2] = {(uint64_t)heads * pra::kD, (uint64_t)rows};
    const uint64_t strides[1] = {(uint64_t)stride * 2};
    return make_tmap_16bit(map, p, 2, dims, strides, box, bf);
  };
  if (!make(&tq, q, q_stride, n_heads, Tq)) return PS_ERR_CUDA;
  if (Tk == 0) {  // no keys at all: no block is ever loaded
    tk = tv = tq;
  } else if (!make(&tk, k, k_stride, n_kv_heads, Tk) || !make(&tv, v, v_stride, n_kv_heads, Tk)) {
    return PS_ERR_CUDA;
  }
  pra::Args a{};
  a.out = out;
  a.o_stride = o_stride;
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.n = n_seqs;
  a.Tq = Tq;
  a.Tk = Tk;
  a.n_heads = n_heads;
  a.group = n_heads / n_kv_heads;
  a.bf16 = bf ? 1 : 0;
  a.wide = (reinterpret_cast<uintptr_t>(out) % 32 == 0 && o_stride % 16 == 0) ? 1 : 0;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.status = status;
  cudaStream_t st = (cudaStream_t)stream;
  auto run = [&](auto kernel, int threads, int smem) -> int {
    PS_CUDA_RET(allow_dynamic_smem(kernel, smem));
    PS_CUDA_RET(launch(kernel, dim3((unsigned)grid), dim3(threads), smem, st, tq, tk, tv, a));
    return PS_OK;
  };
  using One = pra::Shape<1>;
  using Two = pra::Shape<2>;
  if (one)
    return bf ? run(pra::prompt_attention_kernel<__nv_bfloat16, 1>, One::kThreads, One::kSmem)
              : run(pra::prompt_attention_kernel<__half, 1>, One::kThreads, One::kSmem);
  return bf ? run(pra::prompt_attention_kernel<__nv_bfloat16, 2>, Two::kThreads, Two::kSmem)
            : run(pra::prompt_attention_kernel<__half, 2>, Two::kThreads, Two::kSmem);
}
