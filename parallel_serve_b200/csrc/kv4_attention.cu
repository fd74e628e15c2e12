// Decode attention over the 4-bit KV cache (format: kv4.cuh), grouped heads,
// contiguous or paged, both models in one launch.
//
// For one (token, KV head) the G query heads share the cached rows, so a row is
// read once for up to 8 heads and both products run on mma.sync.m16n8k16 (fp16
// inputs, fp32 sums), the 8 heads being the narrow N dimension:
//   S[pos, head] = K[pos, ch] q[ch, head]         M = 16 positions
//   O[ch, head]  = V^T[ch, pos] P[pos, head]      M = 16 channels
// tcgen05 has nothing to offer here: its M is at least 64 rows of an operand in
// shared memory, and the codes have to pass through registers to become 16-bit.
//
// Codes are never converted. A nibble masked in place inside a 16-bit lane is
// the fp16 subnormal c * 2^-24 (bits 0..3) or c * 2^-20 (bits 4..7), exactly, so
// 8 codes cost one shift and four ANDs; the factor 16 between the two is taken
// by q (low-nibble channels times 16) and, for V, by the output channel. Scale
// and zero stay outside the products, in fp32:
//   S = sum_g s_g * (sum_{ch in g} q c) + z_g * (sum_{ch in g} q)
//   O = sum_pos (P s_g) (c - 8)  (P s_g inv_g rounded to fp16)
//       + sum_pos P (z_g + 8 s_g)  (fp32)
// with inv_g a power of two for each group that keeps every s_g inv_g seen at 2^7 or
// less, rescaled like the softmax's running maximum, so bf16 scales of any exponent
// fit and no group's depend on another's. The - 8 (one packed
// subtraction of subnormals, exact) keeps the summands of O as small as the values
// themselves: around c alone, the rounding of P s_g weighs about twice as much and a
// long sum loses the digits that z then cancels.
// P is at most 2^8, so P s_g inv_g fits fp16; one below 2^-14 is a subnormal, off by at
// most 2^-25 of its own 1 / inv_g, which is 2^-31 of the group's largest scale.
// The z term of S is a product too: the sums of q, cut into 16-bit parts that
// together carry fp32's digits, against the stored zeros. q is scaled per head by a
// power of two into fp16's range (exact down to 2^-24 of the head's largest).
//
// S comes out of the instruction with positions in lanes and heads in registers,
// P has to go in with heads in lanes: movmatrix transposes 8 x 8 tiles in
// registers, so P never touches shared memory.
//
// Work: the (token, KV head, block of 8 heads, tile of 128 positions) space is
// cut into equal contiguous ranges over one wave of CTAs from the device's own
// lengths (a captured graph follows them). A producer warp streams tiles through
// an mbarrier ring by bulk copies, 4 compute warps take 32 positions of each. The
// last CTA to finish a piece of an item merges the pieces in order, so results
// do not depend on timing.
//
// 64 sequences of 2048 positions, 32 heads: 164 to 168 us on different GPUs, 4.0 to 4.1 TB/s
// (the bytes alone 102 us at the measured copy rate; loads without arithmetic take
// 109, with the K side 117). One power of two for all groups' scales saves 3 us of it (161
// and 164), and loses the unlikely keys of a group whose scales are far below another's.
// Instructions bound it, and their costs add up: per SM sub-partition a product takes
// 8 cycles and an AND or shift 2, so that unpacking costs as much as multiplying.
// Measured and not kept (beside 161 us, with one power of two): two CTAs of one SM with the same stages (161 us), a ring per
// warp without a producer (193; with four CTAs 252), q in registers (no gain), the - 8
// as a second product with a constant operand (177), tcgen05 products over tiles
// unpacked into shared memory (192 with two CTAs, 211 with three: unpacked, a tile
// takes three times the shared-memory traffic, and its steps wait on one another).
#include <cuda_runtime.h>

#include <type_traits>

#include "kv4.cuh"
#include "ps_host.h"

namespace ps {
namespace kv4 {

constexpr int kHB = 8;                       // query heads of one item
constexpr int kWarps = 4;                    // compute warps
constexpr int kWarpPos = 32;                 // positions of a tile per compute warp
constexpr int kTile = kWarps * kWarpPos;     // 128
constexpr int kStages = 2;
constexpr int kCtasPerSm = 3;
constexpr int kSmallPage = 32;               // positions
constexpr int kAttnThreads = (kWarps + 1) * 32;
constexpr int kTileCodes = kTile * kCodeBytes;
constexpr int kTileMeta = kTile * kMetaBytes;
constexpr int kStageBytes = 2 * (kTileCodes + kTileMeta);  // K codes, K meta, V codes, V meta
constexpr int kMaxEntries = 1024;            // prefix-sum entries of the token lengths
constexpr int kMergeBytes = kWarps * kHB * (kD + 2) * 4;
constexpr int kQBytes = kWarps * 32 * 64;    // q as matrix operand, per warp
constexpr size_t kCounterBytes = 4096;       // arrival counters, zero at rest: one per CTA
constexpr int kAttnSmem = kStages * kStageBytes + kMergeBytes + 256 + kQBytes + (kMaxEntries + 1) * 4;

struct AttnArgs {
  const void* q;  // [M, n_heads, 128], token stride q_stride
  void* out;      // [M, n_heads * 128]
  long long q_stride;
  Pool pool[2];
  const int32_t* pos;
  const int32_t* rows;  // slot or block-table row of token j (nullable)
  const int32_t* counts;
  const int32_t* block_table;
  float* ws_o;   // [2 per CTA][8][128]
  float* ws_ml;  // [2 per CTA][8][2]
  int32_t* counter;
  int32_t* status;
  int split_point, M, n_heads, n_kv, group, hblocks, max_len;
  int L_cap, page_size, page_shift, max_pages, table_rows;
  int per_entry;  // tokens per prefix-sum entry
  float scale_log2;
};

// d += a b on one 16 x 8 x 16 tile; kBf16: bf16 operands, else fp16.
template <bool kBf16 = false>
PS_DEV void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                     uint32_t b0, uint32_t b1) {
  if (kBf16)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = a b (the zero addend costs no register).
template <bool kBf16 = false>
PS_DEV void mma16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                          uint32_t b0, uint32_t b1) {
  if (kBf16)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// 2^x; results below 2^-126 are 0.
PS_DEV float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

PS_DEV void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src)
               : "memory");
}
// One of the barrier's arrivals, when this thread's copies above have landed.
PS_DEV void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

PS_DEV uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Maxima of two pairs of 16-bit values.
template <typename T>
PS_DEV uint32_t max16x2(uint32_t a, uint32_t b) {
  if (std::is_same<T, __half>::value) {
    const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a),
                              *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                   *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}

// a - b of two pairs of fp16 values (exact for codes and 8: subnormals).
PS_DEV uint32_t centre(uint32_t a, uint32_t b) {
  const __half2 d =
      __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&d);
}

PS_DEV uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Cached positions of token j, 0 when its position or home is out of range.
PS_DEV int token_len(const AttnArgs& a, int j, int c0) {
  const int p = a.pos[j];
  const int m = j >= c0 ? 1 : 0;
  const int home = a.rows ? a.rows[j] : (a.block_table ? j : j - (m ? c0 : 0));
  const int cap = a.block_table ? a.max_pages * a.page_size : a.L_cap;
  const int pool_rows = m ? a.pool[1].rows : a.pool[0].rows;
  const bool ok = p >= 0 && p < a.max_len && p < cap && home >= 0 && pool_rows > 0 &&
                  home < (a.block_table ? a.table_rows : pool_rows);
  return ok ? p + 1 : 0;
}

PS_DEV int tiles_of(int len) { return (len + kTile - 1) / kTile; }

// One piece of a CTA's range [b S, b S + S) of tiles: tiles [t0, t1) of item
// (token j, KV head kvh, head block hb), which starts at tile number `start`.
struct Piece {
  int j, len, kvh, hb, t0, t1, start, nt, end;
};

PS_DEV Piece piece_at(const AttnArgs& a, const int32_t* first, int entries, int c0, int g,
                      int g1) {
  const int HB = a.n_kv * a.hblocks;
  int lo = 0, hi = entries - 1;  // last entry that starts at or before g
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] * HB <= g) lo = mid; else hi = mid - 1;
  }
  int at = first[lo] * HB;
  int j = lo * a.per_entry, len = token_len(a, j, c0);
  while (at + tiles_of(len) * HB <= g && j + 1 < a.M) {  // within the entry
    at += tiles_of(len) * HB;
    len = token_len(a, ++j, c0);
  }
  Piece p;
  p.j = j;
  p.len = len;
  p.nt = max(1, tiles_of(len));
  const int it = (g - at) / p.nt;
  p.kvh = it / a.hblocks;
  p.hb = it - p.kvh * a.hblocks;
  p.start = at + it * p.nt;
  p.t0 = g - p.start;
  p.end = min(g1, p.start + p.nt);
  p.t1 = p.end - p.start;
  return p;
}

// One CTA: its range of tiles, piece by piece. Warps 0 to 3 compute, warp 4 loads.
template <typename T>
__global__ void __launch_bounds__(kAttnThreads, kCtasPerSm)
    kv4_decode_attention_kernel(const AttnArgs a) {
  // no pointer arithmetic through integers here: the compiler then knows that
  // every access below is to shared memory (generic loads cost 10% of the time: 193 and 178 us)
  extern __shared__ __align__(128) uint8_t smem[];
  float* so = reinterpret_cast<float*>(smem + kStages * kStageBytes);  // [warp][head][128]
  float* sml = so + kWarps * kHB * kD;                                 // [warp][head][2]
  uint64_t* full = reinterpret_cast<uint64_t*>(sml + kWarps * kHB * 2);
  uint64_t* empty = full + kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + kStages);
  volatile int* last_flag = abort_flag + 1;
  volatile int* stage_bad = last_flag + 1;                         // [kStages]
  int* wsum = const_cast<int*>(stage_bad) + kStages;               // [8]
  // [warp][4 groups]: inv, the scales' power of two (in registers it would spill)
  float4* sinv = reinterpret_cast<float4*>(smem + kStages * kStageBytes + kMergeBytes + 128);
  uint4* sq = reinterpret_cast<uint4*>(smem + kStages * kStageBytes + kMergeBytes + 256);
  int32_t* P =
      reinterpret_cast<int32_t*>(smem + kStages * kStageBytes + kMergeBytes + 256 + kQBytes);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  const int c0 = a.counts ? a.counts[0] : a.split_point;

  // With short pages the (s, z) rows come by 16-byte copies of the producer's lanes:
  // half as many bulk copies, whose number a tile then waits for (pages of 16: 299 and
  // 280 us for 96 ragged sequences, 267 since the producer's addresses are made once a
  // piece: its instructions are taken from the compute warps'; pages of 64: 170 with
  // bulk copies, 174 with these; the codes by 16-byte copies too: 332).
  const bool small_pages = a.block_table && a.page_size <= kSmallPage;

  // Tiles per entry of tokens, then their prefix sums.
  const int entries = (a.M + a.per_entry - 1) / a.per_entry;
  for (int e = tid; e < entries; e += kAttnThreads) {
    int n = 0;
    for (int j = e * a.per_entry; j < min(a.M, (e + 1) * a.per_entry); ++j) {
      const int len = token_len(a, j, c0);
      if (len == 0 && b == 0) set_status(a.status, PS_ERR_BAD_INDEX);
      n += tiles_of(len);
    }
    P[e + 1] = n;
  }
  if (tid == 0) {
    P[0] = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + i, small_pages ? 33 : 1);
      mbar_init(empty + i, kWarps);
    }
    abort_flag[0] = 0;
    fence_mbar_init();
  }
  __syncthreads();
  {
    const int per = (entries + kAttnThreads - 1) / kAttnThreads;
    const int e0 = min(entries, tid * per), e1 = min(entries, e0 + per);
    int run = 0;
    for (int e = e0; e < e1; ++e) run += P[e + 1];
    int incl = run;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    int acc = incl - run;
    for (int w = 0; w < warp; ++w) acc += wsum[w];
    __syncthreads();
    for (int e = e0; e < e1; ++e) {
      acc += P[e + 1];
      P[e + 1] = acc;
    }
  }
  __syncthreads();
  const int W = P[entries] * a.n_kv * a.hblocks;
  const int S = (W + gridDim.x - 1) / gridDim.x;
  const int g0 = min(W, b * S);
  const int g1 = min(W, g0 + S);
  if (g0 >= g1) return;

  if (warp == kWarps) {
    // -------------------------------------------------------------- producer
    const uint64_t pol = l2_policy_evict_first();
    int gs = 0;
    bool dead = false;
    for (int g = g0; g < g1 && !dead;) {
      const Piece pc = piece_at(a, P, entries, c0, g, g1);
      const int m = pc.j >= c0 ? 1 : 0;
      const Pool pool = m ? a.pool[1] : a.pool[0];
      const int home = a.rows ? a.rows[pc.j] : (a.block_table ? pc.j : pc.j - (m ? c0 : 0));
      // paged: the token's table row, the log of a run's positions, row 0 of this head in
      // a page, and rows from one page to the next
      const int32_t* table = a.block_table + (a.block_table ? (size_t)home * a.max_pages : 0);
      const int run_shift = min(a.page_shift, 7);
      const size_t head_row = (size_t)pc.kvh * a.page_size;
      const size_t page_rows = (size_t)a.n_kv * a.page_size;
      const size_t meta_at = (head_row + (lane & (a.page_size - 1))) * kMetaBytes;  // short pages
      for (int t = pc.t0; t < pc.t1; ++t, ++gs) {
        const int st = gs % kStages;
        const int pos0 = t * kTile;
        const int npos = min(kTile, pc.len - pos0);
        // one run per page (128 % page_size == 0 or page_size % 128 == 0, so runs
        // start at multiples of page_size or fill the tile): lane l takes run l (at
        // most 16 of them), and looks its page up while the stage is still in use
        const int o = lane << run_shift;  // the run's first position in the tile
        int page = 0;
        if (a.block_table && o < npos) page = table[(pos0 + o) >> a.page_shift];
        if (!mbar_wait(empty + st, ((gs / kStages) & 1) ^ 1, a.status)) abort_flag[0] = 1;
        dead = __any_sync(0xffffffffu, abort_flag[0] != 0);
        if (dead) break;
        uint8_t* buf = smem + st * kStageBytes;
        if (!a.block_table) {
          if (lane == 0) {
            stage_bad[st] = 0;
            mbar_arrive_expect_tx(full + st, (uint32_t)npos * 2 * (kCodeBytes + kMetaBytes));
          }
          __syncwarp();
          const size_t row = ((size_t)home * a.n_kv + pc.kvh) * a.L_cap + pos0;
          if (lane == 0)
            bulk_load(buf, pool.k_codes + row * kCodeBytes, npos * kCodeBytes, full + st, pol);
          if (lane == 1)
            bulk_load(buf + kTileCodes, pool.k_meta + row * kMetaBytes, npos * kMetaBytes,
                      full + st, pol);
          if (lane == 2)
            bulk_load(buf + kTileCodes + kTileMeta, pool.v_codes + row * kCodeBytes,
                      npos * kCodeBytes, full + st, pol);
          if (lane == 3)
            bulk_load(buf + 2 * kTileCodes + kTileMeta, pool.v_meta + row * kMetaBytes,
                      npos * kMetaBytes, full + st, pol);
        } else {
          bool bad = page < 0 || page >= pool.rows;  // lanes without a run have page 0
          if (bad) page = 0;  // read a page that exists; the piece's output is dropped
          const bool any_bad = __any_sync(0xffffffffu, bad);
          if (lane == 0) {
            if (any_bad) set_status(a.status, PS_ERR_BAD_INDEX);
            stage_bad[st] = any_bad ? 1 : 0;
            mbar_arrive_expect_tx(full + st, (uint32_t)npos * 2 *
                                                 (kCodeBytes + (small_pages ? 0 : kMetaBytes)));
          }
          __syncwarp();
          if (o < npos) {
            const int n = min(1 << run_shift, npos - o);
            const size_t row = page * page_rows + head_row + ((pos0 + o) & (a.page_size - 1));
            bulk_load(buf + o * kCodeBytes, pool.k_codes + row * kCodeBytes, n * kCodeBytes,
                      full + st, pol);
            bulk_load(buf + kTileCodes + kTileMeta + o * kCodeBytes,
                      pool.v_codes + row * kCodeBytes, n * kCodeBytes, full + st, pol);
            if (!small_pages) {
              bulk_load(buf + kTileCodes + o * kMetaBytes, pool.k_meta + row * kMetaBytes,
                        n * kMetaBytes, full + st, pol);
              bulk_load(buf + 2 * kTileCodes + kTileMeta + o * kMetaBytes,
                        pool.v_meta + row * kMetaBytes, n * kMetaBytes, full + st, pol);
            }
          }
          if (small_pages) {
#pragma unroll
            for (int i = 0; i < kTile / 32; ++i) {
              const int r = lane + 32 * i;
              const int pg = __shfl_sync(0xffffffffu, page, r >> a.page_shift);
              if (r < npos) {
                const size_t at = meta_at + pg * (page_rows * kMetaBytes);
                cp_async16(buf + kTileCodes + r * kMetaBytes, pool.k_meta + at);
                cp_async16(buf + 2 * kTileCodes + kTileMeta + r * kMetaBytes, pool.v_meta + at);
              }
            }
            cp_async_arrive(full + st);
          }
        }
      }
      __syncwarp();
      g = pc.end;
    }
    if (dead && lane == 0) {  // let every issued copy land before the CTA exits
      for (int st = 0; st < kStages && st < gs; ++st) {
        const int last = st + kStages * ((gs - 1 - st) / kStages);
        mbar_wait(full + st, (last / kStages) & 1, a.status);
      }
    }
    return;
  }

  // ---------------------------------------------------------------- compute
  const int gr = lane >> 2, t4 = lane & 3;
  // Row gr of a 16-position tile is position sig(gr) of its 8: pairs (2i, 2i+1)
  // keep their places up to order, and rows 0, 2, 4, 6 alternate between even
  // and odd positions, which halves the bank conflicts of the V reads.
  const int sig = gr ^ ((gr >> 1) & 1);
  const int sig0 = (2 * t4) ^ (t4 & 1), sig1 = (2 * t4 + 1) ^ (t4 & 1);
  const uint32_t vsel = (gr & 1) ? 0x7632u : 0x5410u;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  // 8 on the scale of a low and of a high nibble, twice
  constexpr uint32_t kLow8 = 0x00080008u, kHigh8 = 0x00800080u;
  int gs = 0;
  bool dead = false;
  for (int g = g0; g < g1;) {
    const Piece pc = piece_at(a, P, entries, c0, g, g1);
    const int nh = min(kHB, a.group - pc.hb * kHB);
    const int head0 = pc.kvh * a.group + pc.hb * kHB;
    const T* qrow = reinterpret_cast<const T*>(a.q) + (size_t)pc.j * a.q_stride;

    // q as B fragments: lane (gr, t4) holds head gr, channels 32 g + 8 t4 + i,
    // kept in shared memory [group][lane] as (i=0,4) (1,5) (2,6) (3,7): 16
    // registers that the accumulators need more.
    uint4* qb = sq + warp * 128 + lane;
    uint32_t zb[2];        // the groups' sums of q, cut into parts (see below)
    float qf[2];           // the scale of head 2 t4, 2 t4 + 1: softmax scale x its power of two
    {
      uint4 raw[4];
      const bool live = gr < nh;
#pragma unroll
      for (int gi = 0; gi < 4; ++gi)
        raw[gi] = live ? *reinterpret_cast<const uint4*>(qrow + (size_t)(head0 + gr) * kD +
                                                         gi * kGroup + 8 * t4)
                       : make_uint4(0, 0, 0, 0);
      float mx = 0.f, sum[4];
#pragma unroll
      for (int gi = 0; gi < 4; ++gi) {
        const uint32_t u[4] = {raw[gi].x, raw[gi].y, raw[gi].z, raw[gi].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x, y;
          unpack2<T>(u[i], x, y);
          mx = fmaxf(mx, fmaxf(fabsf(x), fabsf(y)));
        }
      }
#pragma unroll
      for (int o = 1; o <= 2; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      // max |q| in [2^e, 2^(e+1)), as far as 2^e and 2^-e are normal numbers (at 2^127 q
      // comes to less than 4 and at bf16's subnormals to less than 1)
      const int e = max(-126, min(126, (int)(__float_as_uint(mx) >> 23) - 127));
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int gi = 0; gi < 4; ++gi) {
        const uint32_t u[4] = {raw[gi].x, raw[gi].y, raw[gi].z, raw[gi].w};
        float f[8];
        sum[gi] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          unpack2<T>(u[i], f[2 * i], f[2 * i + 1]);
          f[2 * i] *= down;
          f[2 * i + 1] *= down;
          sum[gi] += f[2 * i] + f[2 * i + 1];
        }
        // low nibbles: even channels
        qb[gi * 32] = make_uint4(half2_bits(f[0] * 16.f, f[4] * 16.f), half2_bits(f[1], f[5]),
                                 half2_bits(f[2] * 16.f, f[6] * 16.f), half2_bits(f[3], f[7]));
      }
#pragma unroll
      for (int o = 1; o <= 2; o <<= 1)
#pragma unroll
        for (int gi = 0; gi < 4; ++gi) sum[gi] += __shfl_xor_sync(0xffffffffu, sum[gi], o);
      // B operand of the z term: rows k = 4 part + group hold the parts of the
      // group sums, each part what the ones before leave of it in 16 bits
      // (fp16: 11 bits each, bf16: 8; three parts make fp32's 24)
      float r0 = t4 & 1 ? sum[2] : sum[0], r1 = t4 & 1 ? sum[3] : sum[1];
      uint32_t part[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        part[i] = pack2<T>(r0, r1);
        float x, y;
        unpack2<T>(part[i], x, y);
        r0 -= x;
        r1 -= y;
      }
      zb[0] = t4 & 2 ? part[1] : part[0];
      zb[1] = t4 & 2 ? part[3] : part[2];
      const float up = __uint_as_float((uint32_t)(127 + e) << 23) * a.scale_log2;
#pragma unroll
      for (int x = 0; x < 2; ++x)  // from a lane of head 2 t4 + x
        qf[x] = __shfl_sync(0xffffffffu, up, (2 * t4 + x) * 4);
    }

    float o[8][4];   // [2 g + half][channel pair x head]: see the store below
    float zs[4][2];  // sum over positions of P z_g (this lane's rows)
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
    if (lane == 0) {
      const float most = __uint_as_float(253u << 23);  // 2^126
      sinv[warp] = make_float4(most, most, most, most);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
#pragma unroll
    for (int gi = 0; gi < 4; ++gi) zs[gi][0] = zs[gi][1] = 0.f;
    bool bad = false;

    for (int t = pc.t0; t < pc.t1 && !dead; ++t, ++gs) {
      const int st = gs % kStages;
      const bool got = !abort_flag[0] && mbar_wait(full + st, (gs / kStages) & 1, a.status);
      if (!__all_sync(0xffffffffu, got)) {
        abort_flag[0] = 1;
        dead = true;
        break;
      }
      bad |= stage_bad[st] != 0;
      const int left = pc.len - t * kTile - warp * kWarpPos;  // live positions of this warp
      if (left > 0) {
        uint8_t* kc = smem + st * kStageBytes + warp * kWarpPos * kCodeBytes;
        uint8_t* km = smem + st * kStageBytes + kTileCodes + warp * kWarpPos * kMetaBytes;
        uint8_t* vc = kc + kTileCodes + kTileMeta;
        uint8_t* vm = km + kTileCodes + kTileMeta;
        if (left < kWarpPos) {
          // rows behind the last position may hold anything: their scales and
          // zeros become 0 here, their scores -inf below
          if (lane >= left) {
            *reinterpret_cast<uint4*>(km + lane * kMetaBytes) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(vm + lane * kMetaBytes) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();  // before the stage's next bulk copies
          __syncwarp();
        }
        float s[2][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const int r0 = mt * 16 + sig, r1 = r0 + 8;
          const uint4 w0 = *reinterpret_cast<const uint4*>(kc + r0 * kCodeBytes + t4 * 16);
          const uint4 w1 = *reinterpret_cast<const uint4*>(kc + r1 * kCodeBytes + t4 * 16);
          const uint4 e0 = *reinterpret_cast<const uint4*>(km + r0 * kMetaBytes);
          const uint4 e1 = *reinterpret_cast<const uint4*>(km + r1 * kMetaBytes);
          const uint32_t a0[4] = {w0.x, w0.y, w0.z, w0.w}, a1[4] = {w1.x, w1.y, w1.z, w1.w};
          const uint32_t p0[4] = {e0.x, e0.y, e0.z, e0.w}, p1[4] = {e1.x, e1.y, e1.z, e1.w};
          // z term: A row = the position's zeros, pair (0, 1) or (2, 3) in lane t4
          const uint32_t z0 = __byte_perm(t4 & 1 ? e0.z : e0.x, t4 & 1 ? e0.w : e0.y, 0x7632);
          const uint32_t z1 = __byte_perm(t4 & 1 ? e1.z : e1.x, t4 & 1 ? e1.w : e1.y, 0x7632);
          float zt[4], c[4][4], qk[4] = {0.f, 0.f, 0.f, 0.f};
          mma16816_zero<kBf16>(zt, z0, z1, z0, z1, zb[0], zb[1]);
#pragma unroll
          for (int gi = 0; gi < 4; ++gi) {
            const uint32_t h0 = a0[gi] >> 8, h1 = a1[gi] >> 8;
            const uint4 qf4 = qb[gi * 32];
            mma16816_zero(c[gi], a0[gi] & 0x000f000fu, a1[gi] & 0x000f000fu, a0[gi] & 0x00f000f0u,
                          a1[gi] & 0x00f000f0u, qf4.x, qf4.y);
            mma16816(c[gi], h0 & 0x000f000fu, h1 & 0x000f000fu, h0 & 0x00f000f0u,
                     h1 & 0x00f000f0u, qf4.z, qf4.w);
          }
#pragma unroll
          for (int gi = 0; gi < 4; ++gi) {
            float s0, s1, unused;
            unpack2<T>(p0[gi], s0, unused);
            unpack2<T>(p1[gi], s1, unused);
            qk[0] += s0 * c[gi][0], qk[1] += s0 * c[gi][1];
            qk[2] += s1 * c[gi][2], qk[3] += s1 * c[gi][3];
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) s[mt][k] = (qk[k] * 1048576.f + zt[k]) * qf[k & 1];
          if (left < kWarpPos) {
            if (r0 >= left) s[mt][0] = s[mt][1] = -INFINITY;
            if (r1 >= left) s[mt][2] = s[mt][3] = -INFINITY;
          }
        }
        // V's meta of this lane's rows, and their largest scale (low halves)
        uint32_t ve[2][2][4], top2[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint4 e =
                *reinterpret_cast<const uint4*>(vm + (mt * 16 + k * 8 + sig) * kMetaBytes);
            ve[mt][k][0] = e.x, ve[mt][k][1] = e.y, ve[mt][k][2] = e.z, ve[mt][k][3] = e.w;
#pragma unroll
            for (int gi = 0; gi < 4; ++gi) top2[gi] = max16x2<T>(top2[gi], ve[mt][k][gi]);
          }
        float4 inv4 = sinv[warp];
        float smax[4], over = 0.f;
#pragma unroll
        for (int gi = 0; gi < 4; ++gi) {
          float unused;
          unpack2<T>(top2[gi] & 0xffffu, smax[gi], unused);
          over = fmaxf(over, smax[gi] * (&inv4.x)[gi]);
        }
        float mx[2] = {fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2])),
                       fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]))};
        // The references move only when a score is 2^8 above its head's, or a
        // scale above its group's: P (at most 2^8) stays within fp16 and sums keep their
        // precision, and most tiles need no exchange between lanes at all.
        if (__any_sync(0xffffffffu, mx[0] > m_run[0] + 8.f || mx[1] > m_run[1] + 8.f ||
                                        over > 128.f)) {
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int off = 4; off <= 16; off <<= 1)
              mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], off));
          float al[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float mn = fmaxf(m_run[x], mx[x]);
            al[x] = mn == -INFINITY ? 1.f : exp2_ftz(m_run[x] - mn);
            m_run[x] = mn;
            l_run[x] *= al[x];
          }
#pragma unroll
          for (int gi = 0; gi < 4; ++gi) {
            // 2^7 / the next power of two above the largest scale of the warp's rows,
            // within normal numbers
            const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(smax[gi])) >> 23;
            const float was = (&inv4.x)[gi];
            const float now = fminf(was, __uint_as_float(min(253u, 260u - top) << 23));
            const float shrink = now * __uint_as_float(0x7f000000u - __float_as_uint(was));
            const float f0 = al[0] * shrink, f1 = al[1] * shrink;
#pragma unroll
            for (int i = 2 * gi; i < 2 * gi + 2; ++i)
              o[i][0] *= f0, o[i][1] *= f1, o[i][2] *= f0, o[i][3] *= f1;
            zs[gi][0] *= al[0], zs[gi][1] *= al[1];
            (&inv4.x)[gi] = now;
          }
          __syncwarp();
          if (lane == 0) sinv[warp] = inv4;
        }
        const float mu[2] = {m_run[0] == -INFINITY ? 0.f : m_run[0],
                             m_run[1] == -INFINITY ? 0.f : m_run[1]};
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          float p[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) p[k] = exp2_ftz(s[mt][k] - mu[k & 1]);
          l_run[0] += p[0] + p[2];
          l_run[1] += p[1] + p[3];
          // V codes of rows 2 t4, 2 t4 + 1 and 2 t4 + 8, 2 t4 + 9
          uint32_t v[4][4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = mt * 16 + (k >> 1) * 8 + ((k & 1) ? sig1 : sig0);
            const uint4 w = *reinterpret_cast<const uint4*>(vc + r * kCodeBytes + (gr >> 1) * 16);
            v[k][0] = w.x, v[k][1] = w.y, v[k][2] = w.z, v[k][3] = w.w;
          }
#pragma unroll
          for (int gi = 0; gi < 4; ++gi) {
            float s0, z0, s1, z1;
            unpack2<T>(ve[mt][0][gi], s0, z0);
            unpack2<T>(ve[mt][1][gi], s1, z1);
            const float w0 = s0 * (&inv4.x)[gi], w1 = s1 * (&inv4.x)[gi];
            const uint32_t b0 = transpose8x8(half2_bits(p[0] * w0, p[1] * w0));
            const uint32_t b1 = transpose8x8(half2_bits(p[2] * w1, p[3] * w1));
            z0 += 8.f * s0;
            z1 += 8.f * s1;
            zs[gi][0] += p[0] * z0 + p[2] * z1;
            zs[gi][1] += p[1] * z0 + p[3] * z1;
            // halfword gr of the group: channels 4 gr + 0..3 of both positions
            const uint32_t x = __byte_perm(v[0][gi], v[1][gi], vsel);
            const uint32_t y = __byte_perm(v[2][gi], v[3][gi], vsel);
            const uint32_t xh = x >> 8, yh = y >> 8;
            mma16816(o[2 * gi], centre(x & 0x000f000fu, kLow8), centre(x & 0x00f000f0u, kHigh8),
                     centre(y & 0x000f000fu, kLow8), centre(y & 0x00f000f0u, kHigh8), b0, b1);
            mma16816(o[2 * gi + 1], centre(xh & 0x000f000fu, kLow8),
                     centre(xh & 0x00f000f0u, kHigh8), centre(yh & 0x000f000fu, kLow8),
                     centre(yh & 0x00f000f0u, kHigh8), b0, b1);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + st);
    }

    // ---- merge the four warps. o[2 gi + x][0..1]: channel 32 gi + 4 gr + 2 x,
    // heads 2 t4, 2 t4 + 1; [2..3]: the next channel (a high nibble).
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) {
        l_run[x] += __shfl_xor_sync(0xffffffffu, l_run[x], off);
#pragma unroll
        for (int gi = 0; gi < 4; ++gi)
          zs[gi][x] += __shfl_xor_sync(0xffffffffu, zs[gi][x], off);
      }
    __syncwarp();
    const float4 inv4 = sinv[warp];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int head = 2 * t4 + x;
      if (gr == 0) {
        sml[(warp * kHB + head) * 2] = m_run[x];
        sml[(warp * kHB + head) * 2 + 1] = l_run[x];
      }
#pragma unroll
      for (int gi = 0; gi < 4; ++gi) {
        const float z = zs[gi][x];
        // 2^24 and 2^20 first: divided by inv they may be beyond fp32
        const float ref = __uint_as_float(0x7f000000u - __float_as_uint((&inv4.x)[gi]));
        float4 f;
        f.x = o[2 * gi][x] * 16777216.f * ref + z;
        f.y = o[2 * gi][2 + x] * 1048576.f * ref + z;
        f.z = o[2 * gi + 1][x] * 16777216.f * ref + z;
        f.w = o[2 * gi + 1][2 + x] * 1048576.f * ref + z;
        *reinterpret_cast<float4*>(so + (warp * kHB + head) * kD + gi * kGroup + 4 * gr) = f;
      }
    }
    dead = named_bar_or(1, kWarps * 32, dead);
    bad |= dead;
    const int ch = tid;
    T* out = reinterpret_cast<T*>(a.out) + ((size_t)pc.j * a.n_heads + head0) * kD + ch;
    // CTAs [cf, cl] have pieces of this item; a CTA's slot 0 is its range's first piece
    const int cf = pc.start / S, cl = (pc.start + pc.nt - 1) / S;
    const size_t slot = (size_t)b * 2 + (g == g0 ? 0 : 1);
    for (int h = 0; h < nh; ++h) {
      float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sml[(w * kHB + h) * 2]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = sml[(w * kHB + h) * 2];
        const float f = mw == -INFINITY ? 0.f : exp2f(mw - M);
        L += sml[(w * kHB + h) * 2 + 1] * f;
        O += so[(w * kHB + h) * kD + ch] * f;
      }
      if (cf == cl) {
        if (!bad) out[h * kD] = from_f32<T>(O / L);
      } else {
        __stcg(a.ws_o + (slot * kHB + h) * kD + ch, O);
        if (ch == 0) {
          __stcg(a.ws_ml + (slot * kHB + h) * 2, M);
          __stcg(a.ws_ml + (slot * kHB + h) * 2 + 1, bad ? -1.f : L);  // l < 0: a bad piece
        }
      }
    }
    named_bar_sync(1, kWarps * 32);
    if (cf != cl) {
      // ranges are contiguous, so at most one item continues past each CTA's
      // end: its first CTA's number identifies it
      int32_t* counter = a.counter + cf;
      if (tid == 0) {
        fence_acq_rel_gpu();
        const int old = atom_add_acq_rel_gpu(counter, 1);
        const int last = old == cl - cf ? 1 : 0;
        if (last) *counter = 0;
        last_flag[0] = last;
      }
      named_bar_sync(1, kWarps * 32);
      if (last_flag[0]) {
        // pieces in CTA order; CTA c's piece of this item is its first unless
        // the item starts inside c's range
        for (int h = 0; h < nh; ++h) {
          float M = -INFINITY, L = 0.f, O = 0.f;
          bool any_bad = false;
#pragma unroll 4
          for (int c = cf; c <= cl; ++c) {
            const size_t sl = (size_t)c * 2 + (pc.start <= c * S ? 0 : 1);
            const float mc = __ldcg(a.ws_ml + (sl * kHB + h) * 2);
            const float lc = __ldcg(a.ws_ml + (sl * kHB + h) * 2 + 1);
            const float oc = __ldcg(a.ws_o + (sl * kHB + h) * kD + ch);
            any_bad |= lc < 0.f;
            const float mn = fmaxf(M, mc);
            const float fa = M == -INFINITY ? 0.f : exp2f(M - mn);
            const float fb = mc == -INFINITY ? 0.f : exp2f(mc - mn);
            L = L * fa + lc * fb;
            O = O * fa + oc * fb;
            M = mn;
          }
          if (!any_bad) out[h * kD] = from_f32<T>(O / L);
        }
      }
    }
    named_bar_sync(1, kWarps * 32);  // so / sml / last_flag are reused
    g = pc.end;
  }
}

struct AttnPlan {
  int grid, per_entry;
  size_t ml_bytes, o_bytes;
  size_t bytes() const { return kCounterBytes + ml_bytes + o_bytes; }
};

// One wave of CTAs, fewer when the longest lengths give fewer tiles.
static AttnPlan plan_attention(int M, int n_kv, int hblocks, int max_len, int device) {
  AttnPlan p;
  const long long tiles = (long long)M * n_kv * hblocks * cdiv(max_len, kTile);
  long long wave = (long long)kCtasPerSm * sm_count(device);
  if (wave > (long long)(kCounterBytes / 4)) wave = kCounterBytes / 4;
  p.grid = (int)(tiles < wave ? tiles : wave);
  p.per_entry = cdiv(M, kMaxEntries);
  p.ml_bytes = ((size_t)p.grid * 2 * kHB * 2 * 4 + 255) / 256 * 256;
  p.o_bytes = (size_t)p.grid * 2 * kHB * kD * 4;
  return p;
}

}  // namespace kv4
}  // namespace ps

using namespace ps;

extern "C" size_t ps_kv4_decode_attention_workspace_bytes(int M, int n_heads, int n_kv_heads,
                                                          int max_len) {
  if (M <= 0 || n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads || max_len <= 0) return 0;
  const kv4::AttnPlan p = kv4::plan_attention(
      M, n_kv_heads, cdiv(n_heads / n_kv_heads, kv4::kHB), max_len, current_device());
  return p.bytes();
}

extern "C" int ps_kv4_decode_attention(const void* q, long long q_stride,
                                       const ps_kv4_cache_t* cache, void* out, const int32_t* pos,
                                       const int32_t* rows, const int32_t* counts,
                                       int split_point, int M, int n_heads, int max_len,
                                       float scale, int dtype, void* workspace,
                                       size_t workspace_bytes, int32_t* status,
                                       ps_stream_t stream) {
  PS_CHECK_ARG(kv4::valid_cache(cache));
  const int n_kv = cache->n_kv_heads;
  PS_CHECK_ARG(M >= 0 && n_heads > 0 && n_heads % n_kv == 0 && max_len > 0);
  PS_CHECK_ARG(max_len <= (cache->block_table ? cache->max_pages * cache->page_size : cache->L_cap));
  PS_CHECK_ARG(dtype == PS_DTYPE_F16 || dtype == PS_DTYPE_BF16);
  PS_CHECK_ARG(scale > -kMaxScale && scale < kMaxScale);  // NaN fails both
  if (!counts) PS_CHECK_ARG(split_point >= 0 && split_point <= M);
  if (M == 0) return PS_OK;
  PS_CHECK_ARG(q && out && pos && aligned16(q) && q_stride >= (long long)n_heads * kv4::kD &&
               q_stride % 8 == 0);
  PS_CHECK_ARG(!cache->block_table || rows || cache->table_rows >= M);
  const int hblocks = cdiv(n_heads / n_kv, kv4::kHB);
  // tile numbers are 32-bit
  if ((long long)M * n_kv * hblocks * cdiv(max_len, kv4::kTile) > (1ll << 30))
    return PS_ERR_UNSUPPORTED;
  const int device = current_device();
  if (!is_sm100(device)) return PS_ERR_UNSUPPORTED;
  const kv4::AttnPlan p = kv4::plan_attention(M, n_kv, hblocks, max_len, device);
  if (!workspace || workspace_bytes < p.bytes()) return PS_ERR_WORKSPACE;
  PS_CHECK_ARG(aligned16(workspace));
  kv4::AttnArgs a{};
  a.q = q;
  a.out = out;
  a.q_stride = q_stride;
  a.pool[0] = kv4::to_pool(&cache->pool[0]);
  a.pool[1] = kv4::to_pool(&cache->pool[1]);
  a.pos = pos;
  a.rows = rows;
  a.counts = counts;
  a.block_table = cache->block_table;
  char* ws = reinterpret_cast<char*>(workspace);
  a.counter = reinterpret_cast<int32_t*>(ws);
  a.ws_ml = reinterpret_cast<float*>(ws + kv4::kCounterBytes);
  a.ws_o = reinterpret_cast<float*>(ws + kv4::kCounterBytes + p.ml_bytes);
  a.status = status;
  a.split_point = split_point;
  a.M = M;
  a.n_heads = n_heads;
  a.n_kv = n_kv;
  a.group = n_heads / n_kv;
  a.hblocks = hblocks;
  a.max_len = max_len;
  a.L_cap = cache->L_cap;
  a.page_size = cache->page_size;
  a.page_shift = 0;
  while (cache->block_table && (1 << a.page_shift) < cache->page_size) ++a.page_shift;
  a.max_pages = cache->max_pages;
  a.table_rows = cache->table_rows;
  a.per_entry = p.per_entry;
  a.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == PS_DTYPE_BF16) {
    PS_CUDA_RET(allow_dynamic_smem(kv4::kv4_decode_attention_kernel<__nv_bfloat16>, kv4::kAttnSmem));
    PS_CUDA_RET(launch(kv4::kv4_decode_attention_kernel<__nv_bfloat16>, dim3(p.grid),
                       dim3(kv4::kAttnThreads), kv4::kAttnSmem, st, a));
  } else {
    PS_CUDA_RET(allow_dynamic_smem(kv4::kv4_decode_attention_kernel<__half>, kv4::kAttnSmem));
    PS_CUDA_RET(launch(kv4::kv4_decode_attention_kernel<__half>, dim3(p.grid),
                       dim3(kv4::kAttnThreads), kv4::kAttnSmem, st, a));
  }
  return PS_OK;
}
