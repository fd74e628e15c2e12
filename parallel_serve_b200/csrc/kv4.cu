// Head norms + position rotation in one pass, the 4-bit cache's write and its
// read-back (format: kv4.cuh). Elementwise work on 128-channel rows: what bounds
// all three is memory traffic, so every row is read once and written once, 16
// bytes a lane.
//
// Half a warp owns a row (lane l of 16: channels 8l .. 8l+7), so the norm's sum
// takes 4 shuffles, the half-layout rotation exchanges with the lane rotary/16
// away (interleaved pairs stay inside a lane), and a 32-channel group is 4
// lanes. A block works on one token; each half warp takes up to kRows of the
// token's heads, issues their loads together and reuses the token's cos / sin.
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
constexpr int kHalfWarps = kThreads / 16;
constexpr int kRows = 4;  // rows of one half warp in the read-back

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
  int rows_per;  // rows of one half warp
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

// Quantise this lane's 8 channels with the 3 other lanes of its group and store
// its word of codes (and the group's (s, z), by its first lane).
//
// The quotient d / s is y = d r with r = 1 / s, corrected once by its own remainder,
// y + (d - s y) r (Markstein's step): the correctly rounded quotient, so that next
// to half-integers (with 16-bit inputs 2 in 1000 are exact halves) the code is the
// one that a division would give. (A division for each
// channel took most of this kernel's time.) Rounding and packing go through the
// low mantissa bits of 1.5 * 2^23 + quotient; a conversion to integer takes four
// times as long.
template <typename T>
PS_DEV void store_row4(const float (&x)[8], int lane, unsigned mask, uint8_t* codes, uint8_t* meta) {
  float lo = x[0], hi = x[0], zero = 0.f;  // zero: NaN when an x is not finite
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    zero = fmaf(x[i], 0.f, zero);
  }
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(mask, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(mask, hi, o));
  }
  const int g = lane >> 2, w = lane & 3;
  const unsigned nonfinite = __ballot_sync(mask, zero != zero);
  const bool bad = (nonfinite >> ((threadIdx.x & 16) + 4 * g)) & 15u;
  T zt = saturate<T>(lo);
  const float z = to_f32<T>(zt);
  const float span = __fsub_rn(hi, z);
  float range = span * (1.f / 15.f);
  range = fmaf(fmaf(-15.f, range, span), 1.f / 15.f, range);
  if (isinf(span)) range = hi / 15.f - z / 15.f;  // max - min beyond fp32
  T st = saturate<T>(range);
  float s = to_f32<T>(st);
  if (s == 0.f) s = 1.f;  // a constant group: every code 0
  uint32_t word = 0;
  if (s < 1.1754944e-38f || isinf(span)) {
    // 1 / s or a difference may not exist in fp32: divide
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      const float y = __fdiv_rn(__fsub_rn(x[i], z), s);
      word = word * 16u + (uint32_t)rintf(fminf(fmaxf(y, 0.f), 15.f));
    }
  } else {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    r = fmaf(r, fmaf(-s, r, 1.f), r);  // to the last bit, which the step below wants
    const uint64_t zz = f32x2(-z, -z), rr = f32x2(r, r), ss = f32x2(-s, -s);
#pragma unroll
    for (int i = 6; i >= 0; i -= 2) {
      const uint64_t d = f32x2_add(f32x2(x[i], x[i + 1]), zz);
      const uint64_t y0 = f32x2_mul(d, rr);
      float lo_y, hi_y;
      f32x2_split(f32x2_fma(f32x2_fma(ss, y0, d), rr, y0), lo_y, hi_y);
      hi_y = __fadd_rn(fminf(fmaxf(hi_y, 0.f), 15.f), 12582912.f);
      lo_y = __fadd_rn(fminf(fmaxf(lo_y, 0.f), 15.f), 12582912.f);
      word = (word * 16u + __float_as_uint(hi_y)) * 16u + __float_as_uint(lo_y);
    }
    word -= 0x3f400000u;  // 0x4b400000 (1 + 16 + 256 + ...) in 32 bits
  }
  if (bad) {
    word = 0;
    st = from_f32<T>(0.f);
    zt = from_f32<T>(__uint_as_float(0x7fc00000u));
  }
  reinterpret_cast<uint32_t*>(codes)[4 * w + g] = word;
  if (w == 0) {
    T pair[2] = {st, zt};
    reinterpret_cast<uint32_t*>(meta)[g] = *reinterpret_cast<uint32_t*>(pair);
  }
}

// grid (M, ceil(rows per token / (kHalfWarps * rows_per))). Rows of a token: its q
// heads, its k heads, then (append) its v heads.
template <typename T, bool kAppend>
__global__ void __launch_bounds__(kThreads, 8) norm_rope_kernel(const RowArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int j = blockIdx.x;
  const int hw = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const unsigned mask = 0xffffu << (threadIdx.x & 16);
  const int nq = a.q ? a.n_heads : 0;
  const int total = nq + (kAppend ? 2 : 1) * a.n_kv;
  const int c0 = a.counts ? a.counts[0] : a.split_point;
  const int m = j >= c0 ? 1 : 0;
  const int p = a.pos[j];
  bool ok = p >= 0 && (!a.rc || p < a.rope_len);
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
  if (!ok) {
    if (threadIdx.x == 0 && blockIdx.y == 0) set_status(a.status, PS_ERR_BAD_INDEX);
    return;
  }
  const int r0 = blockIdx.y * (kHalfWarps * a.rows_per) + hw;
  const T* qj = (const T*)a.q + (size_t)j * a.q_stride;
  const T* kj = (const T*)a.k + (size_t)j * a.k_stride;
  const T* vj = kAppend ? (const T*)a.v + (size_t)j * a.v_stride : nullptr;
  auto load = [&](int r) {  // this lane's 16 bytes of row r (zeros behind the last)
    Vec8 x = {{0u, 0u, 0u, 0u}};
    if (r < total) {
      const T* src = r < nq ? qj + r * kD
                            : (r < nq + a.n_kv ? kj + (r - nq) * kD : vj + (r - nq - a.n_kv) * kD);
      x = reinterpret_cast<const Vec8*>(src)[lane];
    }
    return x;
  };
  Vec8 next = load(r0), after = load(r0 + kHalfWarps);  // two rows ahead
  // cos / sin of this lane's channels: half layout channel i < rotary/2 pairs
  // with i + rotary/2; interleaved pairs are (2i, 2i + 1)
  const int half = a.rotary >> 1;
  const bool turned = a.rc && 8 * lane < a.rotary;
  const int pair0 = a.interleaved ? 4 * lane : (8 * lane < half ? 8 * lane : 8 * lane - half);
  float co[8] = {}, si[8] = {};
  if (turned) {
    const float* rc = a.rc + (size_t)p * half + pair0;
    const float* rs = a.rs + (size_t)p * half + pair0;
    const int n4 = a.interleaved ? 1 : 2;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i < n4) {
        const float4 c4 = reinterpret_cast<const float4*>(rc)[i];
        const float4 s4 = reinterpret_cast<const float4*>(rs)[i];
        co[4 * i] = c4.x, co[4 * i + 1] = c4.y, co[4 * i + 2] = c4.z, co[4 * i + 3] = c4.w;
        si[4 * i] = s4.x, si[4 * i + 1] = s4.y, si[4 * i + 2] = s4.z, si[4 * i + 3] = s4.w;
      }
    }
  }
  const bool upper = 8 * lane >= half;  // the second element of its half-layout pairs
  const int partner = turned ? (upper ? lane - half / 8 : lane + half / 8) : lane;
  if (!a.interleaved && !upper) {
#pragma unroll
    for (int i = 0; i < 8; ++i) si[i] = -si[i];
  }

#pragma unroll 1
  for (int u = 0; u < a.rows_per; ++u) {
    const int r = r0 + u * kHalfWarps;
    if (r >= total) break;  // the same for the whole half warp
    const Vec8 in = next;
    next = after;
    if (u + 2 < a.rows_per) after = load(r + 2 * kHalfWarps);
    const bool is_q = r < nq, is_v = r >= nq + a.n_kv;
    float x[8];
    unpack8<T>(in, x);
    const T* w = (const T*)(is_q ? a.q_w : a.k_w);
    if (!is_v && w) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
      const float rstd = rsqrtf(ss * (1.f / kD) + a.eps);
      float g[8];
      unpack8<T>(reinterpret_cast<const Vec8*>(w + m * kD)[lane], g);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * rstd * g[i];
    }
    if (!is_v && a.rc) {
      if (a.interleaved) {
        if (turned) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = x[2 * i], o = x[2 * i + 1];
            x[2 * i] = __fsub_rn(__fmul_rn(e, co[i]), __fmul_rn(o, si[i]));
            x[2 * i + 1] = __fadd_rn(__fmul_rn(o, co[i]), __fmul_rn(e, si[i]));
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = __shfl_sync(mask, x[i], partner, 16);
          // si is - sin in the first elements of the pairs; the two products are
          // rounded each (a packed mul and add would be contracted to one fma)
          if (turned) x[i] = __fadd_rn(__fmul_rn(x[i], co[i]), __fmul_rn(y, si[i]));
        }
      }
    }
    if (is_q) {
      T* dst = (T*)a.q_out + (size_t)j * a.qo_stride + r * kD;
      reinterpret_cast<Vec8*>(dst)[lane] = pack8<T>(x);
    } else if (!kAppend) {
      T* dst = (T*)a.k_out + (size_t)j * a.ko_stride + (r - nq) * kD;
      reinterpret_cast<Vec8*>(dst)[lane] = pack8<T>(x);
    } else {
      const int h = is_v ? r - nq - a.n_kv : r - nq;
      const size_t row = cache_row + (size_t)h * cache_len;
      store_row4<T>(x, lane, mask, (is_v ? pool.v_codes : pool.k_codes) + row * kCodeBytes,
                    (is_v ? pool.v_meta : pool.k_meta) + row * kMetaBytes);
    }
  }
}

// Read-back: output row r of sequence i (cu[i] <= r < cu[i+1]) is position
// seqs[i].first + (r - cu[i]). grid (ceil(total / 32), n_kv), 8 half warps with
// 4 rows each, whose loads are all issued before the first is used.
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
  const int hw = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int h = blockIdx.y;
  const int base = blockIdx.x * kHalfWarps * kRows + hw;
  if (base >= a.total) return;
  int lo = 0, hi = a.n;  // the last i with cu[i] <= base, or n
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.cu[mid] <= base) lo = mid; else hi = mid - 1;
  }
  const int g = lane >> 2, w = lane & 3;
  // of the current sequence: its rows [begin, end), home, first position, pool
  int i = lo - 1, begin = 0, end = base, home = 0, first = 0;
  bool known = false, good = false;
  Pool pool{};
  size_t src = 0;  // cache row of this lane's row (contiguous: moves with it)
  uint32_t kw[kRows], vw[kRows], km[kRows], vm[kRows];
  unsigned live = 0;
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int r = base + u * kHalfWarps;
    src += kHalfWarps;
    while (end <= r && i + 1 < a.n) {
      ++i;
      begin = a.cu[i];
      end = a.cu[i + 1];
      known = false;
    }
    if (r >= a.total || i < 0 || r < begin || r >= end) continue;  // no sequence's row
    if (!known) {
      const int m = a.seqs[3 * i];
      home = a.seqs[3 * i + 1];
      first = a.seqs[3 * i + 2];
      pool = m == 1 ? a.pool[1] : a.pool[0];
      good = (m == 0 || m == 1) && home >= 0 && first >= 0 &&
             home < (a.block_table ? a.table_rows : pool.rows);
      if (!a.block_table)
        src = ((size_t)home * a.n_kv + h) * a.L_cap + (size_t)((long long)first + r - begin);
      known = true;
    }
    const long long p = (long long)first + r - begin;
    bool ok = good;
    if (a.block_table) {
      const long long page = p >> a.page_shift;
      ok = ok && page < a.max_pages;
      const int row = ok ? a.block_table[(size_t)home * a.max_pages + page] : -1;
      ok = ok && row >= 0 && row < pool.rows;
      src = ((size_t)row * a.n_kv + h) * a.page_size + ((int)p & (a.page_size - 1));
    } else {
      ok = ok && p < a.L_cap;
    }
    if (!ok) {
      if (lane == 0 && h == 0) set_status(a.status, PS_ERR_BAD_INDEX);
      continue;
    }
    live |= 1u << u;
    kw[u] = reinterpret_cast<const uint32_t*>(pool.k_codes + src * kCodeBytes)[4 * w + g];
    vw[u] = reinterpret_cast<const uint32_t*>(pool.v_codes + src * kCodeBytes)[4 * w + g];
    km[u] = reinterpret_cast<const uint32_t*>(pool.k_meta + src * kMetaBytes)[g];
    vm[u] = reinterpret_cast<const uint32_t*>(pool.v_meta + src * kMetaBytes)[g];
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    if (!(live >> u & 1)) continue;
    const size_t dst = ((size_t)(base + u * kHalfWarps) * a.n_kv + h) * kD;
    reinterpret_cast<Vec8*>((T*)a.k_out + dst)[lane] = values8<T>(kw[u], km[u]);
    reinterpret_cast<Vec8*>((T*)a.v_out + dst)[lane] = values8<T>(vw[u], vm[u]);
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

// Rows of a half warp: what a token's rows come to in as few blocks as hold at
// most 6 each (its setup, a table row of cos and sin among it, is shared by them);
// fewer when the tokens alone do not fill the GPU.
static int rows_per_half_warp(int M, int total, int device) {
  const int most = M >= 4 * sm_count(device) ? 6 : 2;
  const int blocks = cdiv(total, kHalfWarps * most);
  return cdiv(total, kHalfWarps * blocks);
}

template <bool kAppend>
static int launch_rows(RowArgs& a, int dtype, cudaStream_t st) {
  const int total = (a.q ? a.n_heads : 0) + (kAppend ? 2 : 1) * a.n_kv;
  a.rows_per = rows_per_half_warp(a.M, total, current_device());
  const dim3 grid(a.M, cdiv(total, kHalfWarps * a.rows_per));
  if (dtype == PS_DTYPE_BF16)
    PS_CUDA_RET(launch(norm_rope_kernel<__nv_bfloat16, kAppend>, grid, dim3(kThreads), 0, st, a));
  else
    PS_CUDA_RET(launch(norm_rope_kernel<__half, kAppend>, grid, dim3(kThreads), 0, st, a));
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
  const dim3 grid(cdiv(total, kv4::kHalfWarps * kv4::kRows), cache->n_kv_heads);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == PS_DTYPE_BF16)
    PS_CUDA_RET(launch(kv4::kv4_gather_kernel<__nv_bfloat16>, grid, dim3(kv4::kThreads), 0, st, a));
  else
    PS_CUDA_RET(launch(kv4::kv4_gather_kernel<__half>, grid, dim3(kv4::kThreads), 0, st, a));
  return PS_OK;
}
