// Rotary positions over several axes (time, height, width of a video token; or one axis, a text's count).
//
// Pair p of a head, (u, v), is turned by the angle  pos[row mod P][axis(p)] * w_p:
//     u' = u cos - v sin      v' = v cos + u sin           (inverse, = the gradient's way back: sin -> -sin)
// The pairs are (p, p + R/2) or, interleaved, (2 p, 2 p + 1) of the first R = 2 * n_pairs values of a head; the others pass through.
//
// Bound: every element is read and written once - HBM.  The angles are formed once per row and pair (64-bit product, one sincospi),
// kept in the LDS and used by all heads of the row: 1 / (2 * heads) of an angle per element.  A workgroup takes ROWS rows so that
// each thread forms about one angle; then 16-byte loads of u and v chunks, one store each.  Plain stores: the attention reads the output
// next.  (Past the caches where they are over 96 MB, a call among calls takes 64 us instead of 67 - 32 clips of 1569 tokens, 308 MB - or 70
// instead of 72 - the 32-bit gradient of four 16-frame clips - but the layer on those 32 clips 249 us instead of 241, on 64 equal.)
#include "rope.h"

namespace oat {

template <class T>
struct RopeArgs {
  const T* x; long long ldx;
  T* out; long long ldo;
  const int* pos; int period;                        // [period, n_axes]
  int M, heads, dim, rows, inverse;
  float2* table;
  OatRope rope;
};

// VEC: every chunk of 16 bytes of u has its partners in one chunk of v (or, interleaved, in itself) and all addresses are multiples
// of 16 bytes; otherwise element by element.
template <class T, bool VEC>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs<T> a) {
  __shared__ float2 cs[1024];                        // rows * n_pairs <= 1024
  constexpr int N = Elem<T>::N;
  typedef typename Elem<T>::v8 V;
  const int np = a.rope.n_pairs, R = 2 * np;
  const int m0 = blockIdx.x * a.rows, nr = min(a.rows, a.M - m0);
  for (int t = threadIdx.x; t < nr * np; t += 256) {
    const int r = t / np, p = t - r * np;
    const int pr = (m0 + r) % a.period;
    const float2 v = rope_cos_sin(a.pos[(size_t)pr * a.rope.n_axes + a.rope.axis[p]], a.rope.turns[p], a.inverse != 0);
    cs[t] = v;
    if (a.table) a.table[(size_t)p * a.M + m0 + r] = v;
  }
  __syncthreads();
  const bool copy = a.out != a.x;
  if constexpr (VEC) {
    // per head: np / N chunks of u with their v (half), or R / N chunks (interleaved); then (dim - R) / N chunks that pass through
    const int turn = a.rope.interleaved ? R / N : np / N, rest = copy ? (a.dim - R) / N : 0, per = turn + rest;
    const int total = nr * a.heads * per;
    for (int t = threadIdx.x; t < total; t += 256) {
      const int rh = t / per, c = t - rh * per, r = rh / a.heads, h = rh - r * a.heads;
      const T* px = a.x + (size_t)(m0 + r) * a.ldx + h * a.dim;
      T* po = a.out + (size_t)(m0 + r) * a.ldo + h * a.dim;
      const float2* w = cs + r * np;
      if (c >= turn) {
        *reinterpret_cast<V*>(po + R + (c - turn) * N) = *reinterpret_cast<const V*>(px + R + (c - turn) * N);
      } else if (a.rope.interleaved) {
        V x = *reinterpret_cast<const V*>(px + c * N);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
          const float2 y = rope_turn((float)x[2 * e], (float)x[2 * e + 1], w[c * (N / 2) + e]);
          x[2 * e] = (T)y.x;
          x[2 * e + 1] = (T)y.y;
        }
        *reinterpret_cast<V*>(po + c * N) = x;
      } else {
        V xu = *reinterpret_cast<const V*>(px + c * N), xv = *reinterpret_cast<const V*>(px + np + c * N);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float2 y = rope_turn((float)xu[e], (float)xv[e], w[c * N + e]);
          xu[e] = (T)y.x;
          xv[e] = (T)y.y;
        }
        *reinterpret_cast<V*>(po + c * N) = xu;
        *reinterpret_cast<V*>(po + np + c * N) = xv;
      }
    }
  } else {
    const int rest = copy ? a.dim - R : 0, per = np + rest;
    const int total = nr * a.heads * per;
    for (int t = threadIdx.x; t < total; t += 256) {
      const int rh = t / per, c = t - rh * per, r = rh / a.heads, h = rh - r * a.heads;
      const T* px = a.x + (size_t)(m0 + r) * a.ldx + h * a.dim;
      T* po = a.out + (size_t)(m0 + r) * a.ldo + h * a.dim;
      if (c >= np) {
        po[R + c - np] = px[R + c - np];
      } else {
        const int iu = a.rope.interleaved ? 2 * c : c, iv = a.rope.interleaved ? 2 * c + 1 : c + np;
        const float2 y = rope_turn((float)px[iu], (float)px[iv], cs[r * np + c]);
        po[iu] = (T)y.x;
        po[iv] = (T)y.y;
      }
    }
  }
}

template <class T>
static int rope_run(const void* x, long long ldx, void* out, long long ldo, const int* pos, int period, int M, int heads, int dim,
                    const OatRope* rope, int inverse, float2* table, hipStream_t s) {
  RopeArgs<T> a{(const T*)x, ldx, (T*)out, ldo, pos, period, M, heads, dim, 0, inverse, table, *rope};
  constexpr int N = Elem<T>::N;
  const int np = rope->n_pairs;
  // about one angle per thread, but no fewer workgroups than four per CU while rows last
  a.rows = max(1, min(256 / np, M / 1024));
  if (M / a.rows >= 1 << 22) a.rows = 1024 / np;                       // (a launch holds 2^32 threads)
  const bool vec = (rope->interleaved ? (2 * np) % N : np % N) == 0 && (dim - 2 * np) % N == 0 && dim % N == 0 && ldx % N == 0 && ldo % N == 0 &&
                   ((uintptr_t)x | (uintptr_t)out) % 16 == 0;
  const int blocks = (int)(((long long)M + a.rows - 1) / a.rows);
  if (blocks >= 1 << 23) { set_error("rope_axes: more rows than a launch can hold (2^23 workgroups)"); return -2; }
  if (vec) OAT_LAUNCH((rope_kernel<T, true>), dim3(blocks), dim3(256), 0, s, a);
  else OAT_LAUNCH((rope_kernel<T, false>), dim3(blocks), dim3(256), 0, s, a);
  return check_launch("rope_axes");
}

int rope_axes(const void* x, long long ldx, void* out, long long ldo, int dtype, const int* pos, int period, int M, int heads, int dim,
              const OatRope* rope, int inverse, float2* table, void* stream) {
  if (M < 0 || heads < 1 || dim < 2) { set_error("rope_axes: no heads, or a head of fewer than two values"); return -1; }
  if (M == 0) return 0;
  if (!x || !out || !pos || !rope) { set_error("rope_axes: x, out, pos and the ladder are needed"); return -1; }
  if (const char* w = rope_wrong(rope, dim)) { set_error(w); return -2; }
  if (period < 1 || M % period) { set_error("rope_axes: the rows are not a whole number of the positions' periods"); return -2; }
  if (ldx < (long long)heads * dim || ldo < (long long)heads * dim) { set_error("rope_axes: a row is shorter than its heads"); return -2; }
  if ((long long)heads * dim > (1 << 20)) { set_error("rope_axes: a row of more than 2^20 values"); return -2; }
  if (x == out && ldx != ldo) { set_error("rope_axes: in place needs one row pitch"); return -2; }
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case 0: return rope_run<bf16>(x, ldx, out, ldo, pos, period, M, heads, dim, rope, inverse, table, s);
    case 1: return rope_run<_Float16>(x, ldx, out, ldo, pos, period, M, heads, dim, rope, inverse, table, s);
    case 2: return rope_run<float>(x, ldx, out, ldo, pos, period, M, heads, dim, rope, inverse, table, s);
  }
  set_error("rope_axes: unknown element type");
  return -2;
}

}  // namespace oat

extern "C" int oat_rope_axes(const void* x, long long ldx, void* out, long long ldo, int dtype, const int* pos, int period, int M,
                             int heads, int dim, const OatRope* rope, int inverse, void* stream) {
  return oat::rope_axes(x, ldx, out, ldo, dtype, pos, period, M, heads, dim, rope, inverse, nullptr, stream);
}
