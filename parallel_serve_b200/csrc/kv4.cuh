// The 4-bit KV cache format shared by the kernels that write it (kv4.cu), read
// it back (kv4.cu) and attend over it (kv4_attention.cu).
//
// A row is the 128 channels of one (position, KV head), cut into 4 groups of 32
// channels. Group g stores (scale s, zero z) in the model's 16-bit type T:
//   z = T(min),  s = T((max - z) / 15),  c = clamp(rint((x - z) / s), 0, 15)
// and stands for s * c + z. z and s are rounded once, to the type that the model
// itself keeps its activations in, so their range covers every value the model
// can produce; the codes are taken against the rounded pair, so that rounding
// only shifts the grid and costs no accuracy of its own. Values that T cannot
// hold saturate; a group with a NaN or an infinity stores s = 0, z = NaN and
// reads back as NaN.
//
// Codes: 64 bytes, 16 words of 8 codes (low nibble first). Word w of group g is
// word 4 * w + g of the row (the 4 x 4 transpose of the natural order): 16
// consecutive bytes then hold one word of every group, which is what a lane of
// the attention's matrix instructions takes in one 16-byte read.
// Meta: 16 bytes, (s, z) of groups 0..3.
#pragma once
#include "ps_common.cuh"

namespace ps {
namespace kv4 {

constexpr int kD = 128;
constexpr int kGroup = 32;
constexpr int kCodeBytes = 64;  // per row
constexpr int kMetaBytes = 16;

// One model's pools: [rows, n_kv, len, 64] codes and [rows, n_kv, len, 4, 2] meta,
// rows = slots (len = L_cap) or pages (len = page_size).
struct Pool {
  uint8_t* k_codes;
  uint8_t* k_meta;
  uint8_t* v_codes;
  uint8_t* v_meta;
  int rows;
};

// Host checks and conversion of the C descriptors (kv4.cu).
bool valid_cache(const ps_kv4_cache_t* c);
Pool to_pool(const ps_kv4_pool_t* p);

template <typename T>
PS_DEV float max_finite();
template <>
PS_DEV float max_finite<__half>() { return 65504.f; }
template <>
PS_DEV float max_finite<__nv_bfloat16>() { return 3.3895313892515355e38f; }

template <typename T>
PS_DEV T saturate(float v) {
  const float m = max_finite<T>();
  return from_f32<T>(fminf(fmaxf(v, -m), m));
}

template <typename T>
PS_DEV uint32_t pack2(float lo, float hi) {
  T v[2] = {from_f32<T>(lo), from_f32<T>(hi)};
  return *reinterpret_cast<uint32_t*>(v);
}

template <typename T>
PS_DEV void unpack2(uint32_t u, float& lo, float& hi) {
  T v[2];
  *reinterpret_cast<uint32_t*>(v) = u;
  lo = to_f32<T>(v[0]);
  hi = to_f32<T>(v[1]);
}
// A bf16 is the upper half of the fp32 of the same value.
template <>
PS_DEV void unpack2<__nv_bfloat16>(uint32_t u, float& lo, float& hi) {
  lo = __uint_as_float(u << 16);
  hi = __uint_as_float(u & 0xffff0000u);
}

}  // namespace kv4
}  // namespace ps
