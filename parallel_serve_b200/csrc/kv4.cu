// Head norms + position rotation in one pass, the 4-bit cache's write and its
// read-back (format: kv4.cuh). Elementwise work on 128-channel rows: what bounds
// all three is memory traffic, so every row is read once and written once, 16
// bytes a lane. (One exception: half-layout pairs of a part of the head lie in different
// lanes, and the other channel's chunk is read a second time, out of L1.)
//
// Norm, rotation and write: four lanes own a row. Lane q has the 16-byte chunks 2q,
// 2q + 1, 2q + 8 and 2q + 9, so both channels of a pair (i, i + 64) of the whole-head
// rotation are in one lane, as interleaved pairs are, and a 32-channel group is two
// lanes: what a group takes beside its channels (its zero, scale and reciprocal)
// is done by two lanes, not by four with four times the calls. Instructions bounded
// the write with 16 lanes to a row: writing and reading back 16 prompts of up to 2048
// tokens with 32 + 32 heads took 575 us, with four lanes for the write 382, with four for
// the read-back, too, 368 (367 to 390 on different GPUs; the bytes alone 299);
// norm and rotation of 16384 tokens with 32 + 8 heads 74 and 63 (52). A block takes a
// few tokens; each quad takes every Q-th of its token's rows, loads one ahead, and
// keeps the token's cos / sin in registers.
// What it reaches now is 5.1 TB/s (append) to 5.5 (norm and rotation alone). Measured and
// not kept: rows three ahead through a shared-memory ring (382 us, write + read 372
// otherwise), 32-byte loads (no change; 32-byte stores: 63 and 61 us), cos / sin read again for each row (61 us
// for norm and rotation alone, ragged write + read 74 instead of 72), fewer registers
// for more warps (386 and more).
//
// Arithmetic is fp32 throughout (norm, weight, rotation, quantisation) with one
// rounding at the end: q / k to the 16-bit type, or straight to codes. The
// rotation's products and sums are rounded separately (no fused multiply-add),
// which keeps x * cos - y * sin symmetric in its two products.
#include <cuda_runtime.h>

#include "kv4.cuh"
#include "ps_host.h"

namespace ps {
namespace kv4 {

constexpr int kThreads = 128;
constexpr int kQuads = kThreads / 4;

struct RowArgs {
  const void* q;  // [M, n_heads, 128], token stride q_stride (elements); nullable
  const void* k;
  const void* v;  // append only
  void* q_out;    // [M, n_heads, 128], token stride
  void* k_out;    // norm + rotation without a cache
  long long q_stride, k_stride, v_stride, qo_stride, ko_stride;
  const void* q_w;  // [2, 128], nullable
  const void* k_w;
  const float* rc;  // [table_len, rotary / 2], nullable
  const float* rs;
  const int32_t* pos;
  const int32_t* rows;         // cache home of token j: slot, or block-table row (nullable)
  const int32_t* counts;       // nullable: split_point
  const int32_t* block_table;  // nullable: contiguous pools
  Pool pool[2];
  int32_t* status;
  int M, n_heads, n_kv, split_point, rotary, interleaved, rope_len;
  int wide;      // q_out and k_out rows are 32-byte aligned
  int quads;     // of a token in a block: a power of two up to kQuads
  int rows_per;  // rows of a quad
  int L_cap, page_size, page_shift, max_pages, table_rows;  // append
  float eps;
};

struct alignas(16) Vec8 {
  uint32_t u[4];
};

template <typename T>
PS_DEV void unpack8(const Vec8& a, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2<T>(a.u[i], f[2 * i], f[2 * i + 1]);
}
template <typename T>
PS_DEV Vec8 pack8(const float* f) {
  Vec8 a;
#pragma unroll
  for (int i = 0; i < 4; ++i) a.u[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
  return a;
}

// Rotations that a kernel is made for: pairs (i, i + 64) of the whole head,
// interleaved pairs, and half-layout pairs of a part of the head.
enum Rotation { kNone, kWhole, kInterleaved, kPart };

// The smallest and largest of three values, NaN when one of them is.
PS_DEV float min3(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
PS_DEV float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Quantise a group: 16 channels of this lane, 16 of the lane beside it. Words of 8
// codes and the group's (s, z).
//
// The quotient d / s is y = d r with r = 1 / s, corrected once by its own remainder,
// y + (d - s y) r (Markstein's step): the correctly rounded quotient, so that next
// to half-integers (with 16-bit inputs 2 in 1000 are exact halves) the code is the
// one that a division would give. A division for each channel took most of this
// kernel's time. Rounding and packing go through the low mantissa bits of
// 1.5 * 2^23 + quotient; a conversion to integer takes four times as long.
template <typename T>
PS_DEV void quantise_group(const float (&a)[8], const float (&b)[8], unsigned mask,
                           uint32_t (&word)[2], uint32_t& meta) {
  float lo = a[0], hi = a[0];  // NaN when one is
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = min3(lo, a[i], b[i]);
    hi = max3(hi, a[i], b[i]);
  }
  const float lo1 = __shfl_xor_sync(mask, lo, 1), hi1 = __shfl_xor_sync(mask, hi, 1);
  lo = min3(lo, lo1, lo1);
  hi = max3(hi, hi1, hi1);
  const bool finite = fabsf(lo) <= 3.402823466e38f && fabsf(hi) <= 3.402823466e38f;
  T zt = saturate<T>(lo);
  const float z = to_f32<T>(zt);
  const float span = __fsub_rn(hi, z);
  float range = span * (1.f / 15.f);
  range = fmaf(fmaf(-15.f, range, span), 1.f / 15.f, range);
  // max - min beyond fp32: differences of halves, whose rounding is the same
  const bool wide = isinf(span);
  const float half = wide ? 0.5f : 1.f;
  if (wide) range = 2.f * __fdiv_rn(__fsub_rn(0.5f * hi, 0.5f * z), 15.f);
  T st = saturate<T>(range);
  float s = to_f32<T>(st);
  if (s == 0.f) s = 1.f;  // a constant group: every code 0
  if (s < 1.1754944e-38f || wide) {
    // 1 / s or a difference may not exist in fp32: divide
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      word[k] = 0;
#pragma unroll
      for (int i = 7; i >= 0; --i) {
        const float y = __fdiv_rn(__fsub_rn(half * (k ? b[i] : a[i]), half * z), half * s);
        word[k] = word[k] * 16u + (uint32_t)rintf(fminf(fmaxf(y, 0.f), 15.f));
      }
    }
  } else {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    r = fmaf(r, fmaf(-s, r, 1.f), r);  // to the last bit, which the step below wants
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      word[k] = 0;
#pragma unroll
      for (int i = 7; i >= 0; --i) {
        const float d = __fsub_rn(k ? b[i] : a[i], z);
        const float y0 = __fmul_rn(d, r);
        const float y = fmaf(fmaf(-s, y0, d), r, y0);
        word[k] = word[k] * 16u +
                  __float_as_uint(__fadd_rn(fminf(fmaxf(y, 0.f), 15.f), 12582912.f));
      }
      word[k] -= 0x3f400000u;  // 0x4b400000 (1 + 16 + 256 + ...) in 32 bits
    }
  }
  if (!finite) {
    word[0] = word[1] = 0;
    st = from_f32<T>(0.f);
    zt = from_f32<T>(__uint_as_float(0x7fc00000u));
  }
  const T pair[2] = {st, zt};
  meta = *reinterpret_cast<const uint32_t*>(pair);
}

// Rows of a token: its q heads, its k heads, then (append) its v heads. grid
// (ceil(M / tokens of a block), row blocks).
template <typename T, bool kAppend, int kRot>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const RowArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int quad = threadIdx.x >> 2, q4 = threadIdx.x & 3;
  const unsigned mask = 0xfu << (threadIdx.x & 28);
  const int j = blockIdx.x * (kQuads / a.quads) + quad / a.quads;
  if (j >= a.M) return;
  const int nq = a.q ? a.n_heads : 0;
  const int total = nq + (kAppend ? 2 : 1) * a.n_kv;
  const int c0 = a.counts ? a.counts[0] : a.split_point;
  const int m = j >= c0 ? 1 : 0;
  const int p = a.pos[j];
  bool ok = p >= 0 && (kRot == kNone || p < a.rope_len);
  size_t cache_row = 0;  // first (row, head 0, position) index of this token
  int cache_len = 0;
  const Pool pool = m ? a.pool[1] : a.pool[0];
  if (kAppend) {
    const int home = a.rows ? a.rows[j] : (a.block_table ? j : j - (m ? c0 : 0));
    ok = ok && home >= 0;
    int at = p, row = home;
    if (a.block_table) {
      cache_len = a.page_size;
      const int page = p >> a.page_shift;
      ok = ok && home < a.table_rows && page < a.max_pages;
      row = ok ? a.block_table[(size_t)home * a.max_pages + page] : -1;
      at = p & (cache_len - 1);
    } else {
      cache_len = a.L_cap;
      ok = ok && p < a.L_cap;
    }
    ok = ok && row >= 0 && row < pool.rows;
    cache_row = ok ? (size_t)row * a.n_kv * cache_len + at : 0;
  }
  const int first = quad % a.quads + blockIdx.y * a.quads * a.rows_per;
  if (!ok) {
    if (first == 0 && q4 == 0) set_status(a.status, PS_ERR_BAD_INDEX);
    return;
  }
  const int last = min(total, (int)(blockIdx.y + 1) * a.quads * a.rows_per);
  const T* qj = (const T*)a.q + (size_t)j * a.q_stride;
  const T* kj = (const T*)a.k + (size_t)j * a.k_stride;
  const T* vj = kAppend ? (const T*)a.v + (size_t)j * a.v_stride : nullptr;
  auto source = [&](int r) {
    return reinterpret_cast<const Vec8*>(
        r < nq ? qj + r * kD : (r < nq + a.n_kv ? kj + (r - nq) * kD : vj + (r - nq - a.n_kv) * kD));
  };
  const int chunk[4] = {2 * q4, 2 * q4 + 1, 2 * q4 + 8, 2 * q4 + 9};
  Vec8 next[4] = {};
  if (first < last) {
    const Vec8* src = source(first);
#pragma unroll
    for (int i = 0; i < 4; ++i) next[i] = src[chunk[i]];
  }
  // cos / sin of this lane's 16 pairs: kWhole, channels 16 q4 + 0 .. 15 and the ones 64
  // above; kInterleaved, 4 of each chunk (cos 1, sin 0 behind the rotary part)
  float co[16], si[16];
  const int half = a.rotary >> 1;
  if (kRot == kWhole || kRot == kInterleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = kRot == kWhole ? 16 * q4 + 4 * i : 4 * chunk[i];
      float4 c4 = make_float4(1.f, 1.f, 1.f, 1.f), s4 = make_float4(0.f, 0.f, 0.f, 0.f);
      if (at < half) {
        c4 = *reinterpret_cast<const float4*>(a.rc + (size_t)p * half + at);
        s4 = *reinterpret_cast<const float4*>(a.rs + (size_t)p * half + at);
      }
      co[4 * i] = c4.x, co[4 * i + 1] = c4.y, co[4 * i + 2] = c4.z, co[4 * i + 3] = c4.w;
      si[4 * i] = s4.x, si[4 * i + 1] = s4.y, si[4 * i + 2] = s4.z, si[4 * i + 3] = s4.w;
    }
  }

#pragma unroll 1
  for (int r = first; r < last; r += a.quads) {
    const Vec8* src = source(r);
    float x[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack8<T>(next[i], x[i]);
    if (r + a.quads < last) {  // one row ahead
      const Vec8* ahead = source(r + a.quads);
#pragma unroll
      for (int i = 0; i < 4; ++i) next[i] = ahead[chunk[i]];
    }
    const bool is_q = r < nq, is_v = r >= nq + a.n_kv;
    const T* w = (const T*)(is_q ? a.q_w : a.k_w);
    float rstd = 1.f;
    if (!is_v && w) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 8; ++c) ss += x[i][c] * x[i][c];
      ss += __shfl_xor_sync(mask, ss, 1);
      ss += __shfl_xor_sync(mask, ss, 2);
      rstd = rsqrtf(ss * (1.f / kD) + a.eps);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float g[8];
        unpack8<T>(reinterpret_cast<const Vec8*>(w + m * kD)[chunk[i]], g);
#pragma unroll
        for (int c = 0; c < 8; ++c) x[i][c] = x[i][c] * rstd * g[c];
      }
    }
    if (kRot != kNone && !is_v) {
      // products and sums are rounded each
      if (kRot == kWhole) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const float e = x[i][c], o = x[i + 2][c], cc = co[8 * i + c], sn = si[8 * i + c];
            x[i][c] = __fsub_rn(__fmul_rn(e, cc), __fmul_rn(o, sn));
            x[i + 2][c] = __fadd_rn(__fmul_rn(o, cc), __fmul_rn(e, sn));
          }
      } else if (kRot == kInterleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * chunk[i] < half) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float e = x[i][2 * c], o = x[i][2 * c + 1];
              const float cc = co[4 * i + c], sn = si[4 * i + c];
              x[i][2 * c] = __fsub_rn(__fmul_rn(e, cc), __fmul_rn(o, sn));
              x[i][2 * c + 1] = __fadd_rn(__fmul_rn(o, cc), __fmul_rn(e, sn));
            }
          }
      } else {
        // pairs (i, i + half) of different lanes: the other channel is read again
        // (a multiple of 8 away, so a whole chunk), before anything is written
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int ch = 8 * chunk[i];
          if (ch < 2 * half) {
            const bool up = ch >= half;
            const int other = up ? chunk[i] - half / 8 : chunk[i] + half / 8;
            float y[8];
            unpack8<T>(src[other], y);
            if (w) {
              float g[8];
              unpack8<T>(reinterpret_cast<const Vec8*>(w + m * kD)[other], g);
#pragma unroll
              for (int c = 0; c < 8; ++c) y[c] = y[c] * rstd * g[c];
            }
            const float* rc = a.rc + (size_t)p * half + (up ? ch - half : ch);
            const float* rs = a.rs + (size_t)p * half + (up ? ch - half : ch);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const float b = __fmul_rn(y[c], rs[c]);
              x[i][c] = __fadd_rn(__fmul_rn(x[i][c], rc[c]), up ? b : -b);
            }
          }
        }
        __syncwarp(mask);
      }
    }
    if (is_q || !kAppend) {
      Vec8* dst = reinterpret_cast<Vec8*>(is_q ? (T*)a.q_out + (size_t)j * a.qo_stride + r * kD
                                               : (T*)a.k_out + (size_t)j * a.ko_stride +
                                                     (r - nq) * kD);
#pragma unroll
      for (int i = 0; i < 4; i += 2) {  // chunks 2 q4 and 2 q4 + 1: 32 bytes
        const Vec8 lo = pack8<T>(x[i]), hi = pack8<T>(x[i + 1]);
        if (a.wide) {
          const uint32_t w[8] = {lo.u[0], lo.u[1], lo.u[2], lo.u[3],
                                 hi.u[0], hi.u[1], hi.u[2], hi.u[3]};
          st_32bytes(dst + chunk[i], w);
        } else {
          dst[chunk[i]] = lo;
          dst[chunk[i + 1]] = hi;
        }
      }
    } else {
      // groups q4 / 2 (chunks 0, 1) and q4 / 2 + 2 (chunks 2, 3): words 2 (q4 & 1)
      // and the next of each
      uint32_t lo[2], hi[2], mlo, mhi;
      quantise_group<T>(x[0], x[1], mask, lo, mlo);
      quantise_group<T>(x[2], x[3], mask, hi, mhi);
      // 16 stored bytes hold one word of every group: exchange with the lane of
      // the two other groups
      const bool up = q4 >> 1;
      const uint32_t r0 = __shfl_xor_sync(mask, up ? lo[0] : lo[1], 2);
      const uint32_t r1 = __shfl_xor_sync(mask, up ? hi[0] : hi[1], 2);
      const int h = is_v ? r - nq - a.n_kv : r - nq;
      const size_t row = cache_row + (size_t)h * cache_len;
      uint8_t* codes = (is_v ? pool.v_codes : pool.k_codes) + row * kCodeBytes;
      uint8_t* meta = (is_v ? pool.v_meta : pool.k_meta) + row * kMetaBytes;
      reinterpret_cast<uint4*>(codes)[2 * (q4 & 1) + (up ? 1 : 0)] =
          up ? make_uint4(r0, lo[1], r1, hi[1]) : make_uint4(lo[0], r0, hi[0], r1);
      if (!(q4 & 1)) {
        reinterpret_cast<uint32_t*>(meta)[q4 >> 1] = mlo;
        reinterpret_cast<uint32_t*>(meta)[(q4 >> 1) + 2] = mhi;
      }
    }
  }
}

// Read-back: output row r of sequence i (cu[i] <= r < cu[i+1]) is position
// seqs[i].first + (r - cu[i]). grid (ceil(total / 32), n_kv). Four lanes to a
// row: lane w reads 16 bytes, word w of every group, for K and for V, and writes the
// 4 x 8 channels of each that they stand for. (One word a lane, 16 lanes to a row,
// takes 4 bytes an instruction and its index arithmetic four times over: ALU at 70%,
// write + read of 16 prompts 382 us; this way 368.)
struct GatherArgs {
  Pool pool[2];
  const int32_t* seqs;  // [n][3]: model, slot or block-table row, first position
  const int32_t* cu;    // [n + 1]
  const int32_t* block_table;
  void* k_out;  // [total, n_kv, 128]
  void* v_out;
  int32_t* status;
  int n, total, n_kv, L_cap, page_size, page_shift, max_pages, table_rows;
};

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  using type = __half2;
  static constexpr uint32_t kBias = 0x64006400u;  // 1024 twice: low mantissa bits are units
};
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static constexpr uint32_t kBias = 0x43004300u;  // 128
};

// The 8 values of a word of codes, two at a time in packed 16-bit arithmetic: a
// nibble placed in the low mantissa bits of a bias is bias + c exactly, and one
// fused s * c + z rounds once.
template <typename T>
PS_DEV Vec8 values8(uint32_t word, uint32_t meta) {
  using T2 = typename Pair<T>::type;
  const uint32_t bias = Pair<T>::kBias, sb = __byte_perm(meta, 0, 0x1010),
                 zb = __byte_perm(meta, 0, 0x3232);
  const T2 s = *reinterpret_cast<const T2*>(&sb), z = *reinterpret_cast<const T2*>(&zb);
  const T2 b = *reinterpret_cast<const T2*>(&bias);
  T top[2] = {from_f32<T>(max_finite<T>()), from_f32<T>(max_finite<T>())};
  Vec8 out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t = word >> (8 * i);
    const uint32_t n = (t & 0xfu) | ((t << 12) & 0xf0000u) | bias;  // low nibble, high nibble
    // 15 s + z may lie half a step of (s, z) above T's largest value; NaN stays
    const T2 v = __hmin2_nan(__hfma2(s, __hsub2(*reinterpret_cast<const T2*>(&n), b), z),
                             *reinterpret_cast<const T2*>(top));
    out.u[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return out;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) kv4_gather_kernel(const GatherArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int w = threadIdx.x & 3, h = blockIdx.y;
  const int r = blockIdx.x * kQuads + (threadIdx.x >> 2);
  if (r >= a.total) return;
  int lo = 0, hi = a.n;  // the last i with cu[i] <= r, or n
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.cu[mid] <= r) lo = mid; else hi = mid - 1;
  }
  if (lo == a.n || r < a.cu[lo]) return;  // no sequence's row
  const int m = a.seqs[3 * lo], home = a.seqs[3 * lo + 1], first = a.seqs[3 * lo + 2];
  const Pool pool = m == 1 ? a.pool[1] : a.pool[0];
  bool ok = (m == 0 || m == 1) && home >= 0 && first >= 0 &&
            home < (a.block_table ? a.table_rows : pool.rows);
  const long long p = (long long)first + r - a.cu[lo];
  size_t src = 0;  // cache row
  if (a.block_table) {
    const long long page = p >> a.page_shift;
    ok = ok && page < a.max_pages;
    const int row = ok ? a.block_table[(size_t)home * a.max_pages + page] : -1;
    ok = ok && row >= 0 && row < pool.rows;
    src = ((size_t)row * a.n_kv + h) * a.page_size + ((int)p & (a.page_size - 1));
  } else {
    ok = ok && p < a.L_cap;
    src = ((size_t)home * a.n_kv + h) * a.L_cap + p;
  }
  if (!ok) {
    if (w == 0 && h == 0) set_status(a.status, PS_ERR_BAD_INDEX);
    return;
  }
  const Vec8 kw = reinterpret_cast<const Vec8*>(pool.k_codes + src * kCodeBytes)[w];
  const Vec8 vw = reinterpret_cast<const Vec8*>(pool.v_codes + src * kCodeBytes)[w];
  const Vec8 km = *reinterpret_cast<const Vec8*>(pool.k_meta + src * kMetaBytes);
  const Vec8 vm = *reinterpret_cast<const Vec8*>(pool.v_meta + src * kMetaBytes);
  const size_t dst = ((size_t)r * a.n_kv + h) * kD;
  Vec8* k = reinterpret_cast<Vec8*>((T*)a.k_out + dst);
  Vec8* v = reinterpret_cast<Vec8*>((T*)a.v_out + dst);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    k[4 * g + w] = values8<T>(kw.u[g], km.u[g]);
    v[4 * g + w] = values8<T>(vw.u[g], vm.u[g]);
  }
}

static bool valid_pool(const ps_kv4_pool_t* p) {
  if (!p || p->rows == 0) return true;
  return p->rows > 0 && p->k_codes && p->k_meta && p->v_codes && p->v_meta &&
         aligned16(p->k_codes) && aligned16(p->k_meta) && aligned16(p->v_codes) &&
         aligned16(p->v_meta);
}

Pool to_pool(const ps_kv4_pool_t* p) {
  Pool r{};
  if (p && p->rows > 0) {
    r.k_codes = (uint8_t*)p->k_codes;
    r.k_meta = (uint8_t*)p->k_meta;
    r.v_codes = (uint8_t*)p->v_codes;
    r.v_meta = (uint8_t*)p->v_meta;
    r.rows = p->rows;
  }
  return r;
}

// Shared checks of the pools and their paging; true when they hold.
bool valid_cache(const ps_kv4_cache_t* c) {
  if (!c || c->n_kv_heads <= 0 || c->n_kv_heads > 65535) return false;
  if (!valid_pool(&c->pool[0]) || !valid_pool(&c->pool[1])) return false;
  if (c->pool[0].rows + (long long)c->pool[1].rows <= 0) return false;
  if (c->block_table) {
    const int ps = c->page_size;
    return ps >= 8 && ps <= 4096 && (ps & (ps - 1)) == 0 && c->max_pages > 0 &&
           c->table_rows > 0 && (long long)c->max_pages * ps <= (1ll << 30);
  }
  return c->L_cap > 0 && c->L_cap <= (1 << 30);
}

template <typename T, bool kAppend>
static cudaError_t launch_rotation(const RowArgs& a, dim3 grid, cudaStream_t st) {
  if (!a.rc) return launch(norm_rope_kernel<T, kAppend, kNone>, grid, dim3(kThreads), 0, st, a);
  if (a.interleaved)
    return launch(norm_rope_kernel<T, kAppend, kInterleaved>, grid, dim3(kThreads), 0, st, a);
  if (a.rotary == kD)
    return launch(norm_rope_kernel<T, kAppend, kWhole>, grid, dim3(kThreads), 0, st, a);
  return launch(norm_rope_kernel<T, kAppend, kPart>, grid, dim3(kThreads), 0, st, a);
}

// How a token's rows are cut: enough quads that each has at most 12 rows (their
// setup, cos and sin among it, is shared by them); one row each, over several
// blocks, when the tokens alone do not fill the GPU.
template <bool kAppend>
static int launch_rows(RowArgs& a, int dtype, cudaStream_t st) {
  auto aligned32 = [](const void* p, long long stride) {
    return reinterpret_cast<uintptr_t>(p) % 32 == 0 && stride % 16 == 0;
  };
  a.wide = aligned32(a.q_out, a.qo_stride) && (kAppend || aligned32(a.k_out, a.ko_stride));
  const int total = (a.q ? a.n_heads : 0) + (kAppend ? 2 : 1) * a.n_kv;
  const bool many = a.M >= 4 * sm_count(current_device());
  const int most = many ? 12 : 1;
  a.quads = 1;
  while (a.quads < kQuads && a.quads * most < total) a.quads *= 2;
  const int blocks = cdiv(total, a.quads * most);
  a.rows_per = cdiv(total, a.quads * blocks);
  const dim3 grid(cdiv(a.M, kQuads / a.quads), blocks);
  PS_CUDA_RET((dtype == PS_DTYPE_BF16 ? launch_rotation<__nv_bfloat16, kAppend>(a, grid, st)
                                      : launch_rotation<__half, kAppend>(a, grid, st)));
  return PS_OK;
}

// The arguments that qk_norm_rope and kv4_append have in common.
static int common_args(RowArgs& a, const void* q, long long q_stride, const void* k,
                       long long k_stride, void* q_out, long long qo_stride, const void* q_w,
                       const void* k_w, float eps, const float* rc, const float* rs, int rope_len,
                       int rotary, int interleaved, const int32_t* pos, const int32_t* counts,
                       int split_point, int M, int n_heads, int n_kv, int dtype,
                       int32_t* status) {
  PS_CHECK_ARG(M >= 0 && n_kv > 0 && n_kv <= 65535);
  PS_CHECK_ARG(dtype == PS_DTYPE_F16 || dtype == PS_DTYPE_BF16);
  if (!counts) PS_CHECK_ARG(split_point >= 0 && split_point <= M);
  PS_CHECK_ARG((rc != nullptr) == (rs != nullptr));
  if (rc)
    PS_CHECK_ARG(rotary > 0 && rotary <= kD && rotary % 16 == 0 && rope_len > 0 && aligned16(rc) &&
                 aligned16(rs));
  PS_CHECK_ARG((q != nullptr) == (q_out != nullptr));
  if (M == 0) return PS_OK;
  PS_CHECK_ARG(k && pos && aligned16(k) && k_stride >= (long long)n_kv * kD && k_stride % 8 == 0);
  if (q)
    PS_CHECK_ARG(n_heads > 0 && n_heads <= 65535 && aligned16(q) && aligned16(q_out) &&
                 q_stride >= (long long)n_heads * kD && q_stride % 8 == 0 &&
                 qo_stride >= (long long)n_heads * kD && qo_stride % 8 == 0);
  PS_CHECK_ARG((!q_w || aligned16(q_w)) && (!k_w || aligned16(k_w)));
  a.q = q;
  a.k = k;
  a.q_out = q_out;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.qo_stride = qo_stride;
  a.q_w = q_w;
  a.k_w = k_w;
  a.rc = rc;
  a.rs = rs;
  a.pos = pos;
  a.counts = counts;
  a.status = status;
  a.M = M;
  a.n_heads = n_heads;
  a.n_kv = n_kv;
  a.split_point = split_point;
  a.rotary = rc ? rotary : 0;
  a.interleaved = interleaved ? 1 : 0;
  a.rope_len = rope_len;
  a.eps = eps;
  return PS_OK;
}

}  // namespace kv4
}  // namespace ps

using namespace ps;

extern "C" int ps_qk_norm_rope(const void* q, long long q_stride, const void* k,
                               long long k_stride, void* q_out, long long qo_stride, void* k_out,
                               long long ko_stride, const void* q_w, const void* k_w, float eps,
                               const float* rope_cos, const float* rope_sin, int rope_len,
                               int rotary_dim, int interleaved, const int32_t* pos,
                               const int32_t* counts, int split_point, int M, int n_heads,
                               int n_kv_heads, int dtype, int32_t* status, ps_stream_t stream) {
  kv4::RowArgs a{};
  const int rc = kv4::common_args(a, q, q_stride, k, k_stride, q_out, qo_stride, q_w, k_w, eps,
                                  rope_cos, rope_sin, rope_len, rotary_dim, interleaved, pos,
                                  counts, split_point, M, n_heads, n_kv_heads, dtype, status);
  if (rc != PS_OK || M == 0) return rc;
  PS_CHECK_ARG(k_out && aligned16(k_out) && ko_stride >= (long long)n_kv_heads * kv4::kD &&
               ko_stride % 8 == 0);
  a.k_out = k_out;
  a.ko_stride = ko_stride;
  return kv4::launch_rows<false>(a, dtype, (cudaStream_t)stream);
}

extern "C" int ps_kv4_append(const void* q, long long q_stride, const void* k, long long k_stride,
                             const void* v, long long v_stride, void* q_out, long long qo_stride,
                             const ps_kv4_cache_t* cache, const void* q_w, const void* k_w,
                             float eps, const float* rope_cos, const float* rope_sin, int rope_len,
                             int rotary_dim, int interleaved, const int32_t* pos,
                             const int32_t* rows, const int32_t* counts, int split_point, int M,
                             int n_heads, int dtype, int32_t* status, ps_stream_t stream) {
  PS_CHECK_ARG(kv4::valid_cache(cache));
  kv4::RowArgs a{};
  const int rc = kv4::common_args(a, q, q_stride, k, k_stride, q_out, qo_stride, q_w, k_w, eps,
                                  rope_cos, rope_sin, rope_len, rotary_dim, interleaved, pos,
                                  counts, split_point, M, n_heads, cache->n_kv_heads, dtype,
                                  status);
  if (rc != PS_OK || M == 0) return rc;
  PS_CHECK_ARG(v && aligned16(v) && v_stride >= (long long)cache->n_kv_heads * kv4::kD &&
               v_stride % 8 == 0);
  PS_CHECK_ARG(!cache->block_table || rows || cache->table_rows >= M);
  a.v = v;
  a.v_stride = v_stride;
  a.rows = rows;
  a.block_table = cache->block_table;
  a.pool[0] = kv4::to_pool(&cache->pool[0]);
  a.pool[1] = kv4::to_pool(&cache->pool[1]);
  a.L_cap = cache->L_cap;
  a.page_size = cache->page_size;
  while (cache->block_table && (1 << a.page_shift) < cache->page_size) ++a.page_shift;
  a.max_pages = cache->max_pages;
  a.table_rows = cache->table_rows;
  return kv4::launch_rows<true>(a, dtype, (cudaStream_t)stream);
}

extern "C" int ps_kv4_gather(const ps_kv4_cache_t* cache, const int32_t* seqs, const int32_t* cu,
                             int n_seqs, int total, void* k_out, void* v_out, int dtype,
                             int32_t* status, ps_stream_t stream) {
  PS_CHECK_ARG(kv4::valid_cache(cache));
  PS_CHECK_ARG(n_seqs >= 0 && total >= 0);
  PS_CHECK_ARG(dtype == PS_DTYPE_F16 || dtype == PS_DTYPE_BF16);
  if (n_seqs == 0 || total == 0) return PS_OK;
  PS_CHECK_ARG(seqs && cu && k_out && v_out && aligned16(k_out) && aligned16(v_out));
  kv4::GatherArgs a{};
  a.pool[0] = kv4::to_pool(&cache->pool[0]);
  a.pool[1] = kv4::to_pool(&cache->pool[1]);
  a.seqs = seqs;
  a.cu = cu;
  a.block_table = cache->block_table;
  a.k_out = k_out;
  a.v_out = v_out;
  a.status = status;
  a.n = n_seqs;
  a.total = total;
  a.n_kv = cache->n_kv_heads;
  a.L_cap = cache->L_cap;
  a.page_size = cache->page_size;
  while (cache->block_table && (1 << a.page_shift) < cache->page_size) ++a.page_shift;
  a.max_pages = cache->max_pages;
  a.table_rows = cache->table_rows;
  const dim3 grid(cdiv(total, kv4::kQuads), cache->n_kv_heads);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == PS_DTYPE_BF16)
    PS_CUDA_RET(launch(kv4::kv4_gather_kernel<__nv_bfloat16>, grid, dim3(kv4::kThreads), 0, st, a));
  else
    PS_CUDA_RET(launch(kv4::kv4_gather_kernel<__half>, grid, dim3(kv4::kThreads), 0, st, a));
  return PS_OK;
}
