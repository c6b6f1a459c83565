// Rotary positions over several axes: the host's description of a ladder and the angle of one pair.
#pragma once
#include "common.h"
#include "../../include/oatrans_hip.h"

namespace oat {

// cos and sin of pos * freq.  The frequency comes as TURNS per position (freq / 2 pi) in 64 bits: the whole turns are dropped there,
// so a far position loses nothing (in 32 bits the angle of position 1e6 would be off by 0.03); what is left lies in [-1/2, 1/2] turns.
OAT_DEV float2 rope_cos_sin(int pos, double turns, bool inverse) {
  const double a = (double)pos * turns;
  const float r = 2.0f * (float)(a - rint(a));
  float s, c;
  sincospif(r, &s, &c);
  return float2{c, inverse ? -s : s};
}

// one pair turned; products and sums are spelt out, so that every kernel rounds alike
OAT_DEV float2 rope_turn(float u, float v, float2 k) {
  return float2{__builtin_fmaf(u, k.x, -(v * k.y)), __builtin_fmaf(v, k.x, u * k.y)};
}

// nullptr, or why a ladder cannot be used for heads of `dim` values
inline const char* rope_wrong(const OatRope* r, int dim) {
  if (r->n_pairs < 1 || r->n_pairs > 64 || 2 * r->n_pairs > dim) return "the ladder has no pair, or more than the head (at most 64)";
  if (r->n_axes < 1 || r->n_axes > 4) return "1 to 4 axes";
  for (int p = 0; p < r->n_pairs; ++p) {
    if (r->axis[p] >= r->n_axes) return "a pair's axis is not one of the ladder's";
    if (!(r->turns[p] >= -1e6 && r->turns[p] <= 1e6)) return "a pair's frequency is not a number, or beyond 1e6 turns";
  }
  return nullptr;
}

// oat_rope_axes; `table` (may be null): the cos and sin of every row's pairs, [n_pairs, M]
int rope_axes(const void* x, long long ldx, void* out, long long ldo, int dtype, const int* pos, int period, int M, int heads, int dim,
              const OatRope* rope, int inverse, float2* table, void* stream);

// a 16-bit or 32-bit element type: vector loads, conversion
template <class T> struct Elem;
template <> struct Elem<bf16> {
  typedef bf16x8 v8;
  static constexpr int N = 8;                       // elements in 16 bytes
};
template <> struct Elem<_Float16> {
  typedef __attribute__((ext_vector_type(8))) _Float16 v8;
  static constexpr int N = 8;
};
template <> struct Elem<float> {
  typedef f32x4 v8;
  static constexpr int N = 4;
};

}  // namespace oat
