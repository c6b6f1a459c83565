// Attention over a sliding window with sinks: forward and backward, ragged sequences, shared key heads.
#include "attn_window.h"

namespace oat {

// ---------------------------------------------------------------------------------------------- forward
// One workgroup = 128 queries of one head, a wave = 32 of them; keys and values pass through the LDS in tiles of 64.
//     S^T = K Q^T      P^T = exp2(c S^T - c m)      O^T += V^T P^T       c = scale log2(e), m = running maximum of the row
// The query is the COLUMN of S^T: a lane holds 16 of 32 keys of ONE query, so maximum and sum of a row are register work and one
// exchange with lane ^ 32, and P^T is the B operand of the second product where it stands.
// Bound: no unit alone, but the way in which two or three waves of a SIMD share them.  Two clips of 7057 tokens (12 heads of 64, window of
// 882 to each side), by counters: the matrix unit is busy 37 % of the time (8 products of 32 clocks per 32 keys of a wave), the vector unit
// 57 % (75 instructions, 16 of them exponentials), the LDS 18 % (4 clocks a KB, no bank conflicts); 2.3 waves are on a SIMD (the registers
// allow 3, the list of tiles is 1.75 rounds of that), and of their time they issue in 42 %, wait to issue in 32 % and for data or the
// barrier in 26 %.  Per 32 keys of a wave that is 700 clocks; in a loop of nothing else the same products take 295, the exponentials, sums
// and conversions 310, both 420 to 440.  Heads of 128 (8191 tokens below): matrix unit 42 %, vector unit 38 %, 1.8 waves.
// Measured (median of 60 runs): the clips 109 us = 660 TFLOP/s; 8191 tokens (32 / 8 heads of 128, causal, window of 1024) 187 us = 691; six
// packed texts of 512 to 2048 (16 / 4 heads of 128, window of 512) 63 us = 435: a fourth of the products there are masked at the window's
// edges, and 1.5 waves are on a SIMD.
// Roundings: P to the operands' 16 bits (pack8); its sum l is of the terms before that, in 32 bits - the terms are off by half a step at most,
// up and down alike.
template <class T, int D>
__global__ __launch_bounds__(256, 2) void win_fwd_kernel(WinArgs a) {
  constexpr int TB = TILE * D * 2;
  __shared__ __attribute__((aligned(1024))) char lds[4 * TB];         // K x 2, V x 2
  const int tiles = (a.max_q + 127) / 128;
  Place pl;
  if (!place(a, tiles, a.Hq, pl)) return;
  const Seq s = load_seq(a, pl.b);
  const int i0 = (tiles - 1 - pl.tile) * 128;                          // causal rows are longest at the end: those first
  if (i0 >= s.nq) {
    if (const int4 t = a.seqs[pl.b]; a.clear && left_out(a, t)) clear_rows<D>(a.out, a.ldo, t.x, t.y, a.rows_q, pl.h, pl.tile, tiles);
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int off = s.nk - s.nq, hk = pl.h / (a.Hq / a.Hkv);
  const KeyTiles kt = key_tiles(a, s.nk, i0 + off, min(i0 + 127, s.nq - 1) + off);
  const char* kb = a.k + (long long)s.k0 * a.ldk + hk * (D * 2);
  const char* vb = a.v + (long long)s.k0 * a.ldv + hk * (D * 2);
  const uint32_t l0 = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) char*)lds);
  const Stager<D> sk(a.ldk), sv(a.ldv);
  auto stage_k = [&](int n, int buf) WIN_INLINE {
    const int j0 = kt.at(n) * TILE;
    sk(kb + (long long)j0 * a.ldk, s.nk - 1 - j0, l0 + buf * TB);
  };
  auto stage_v = [&](int n, int buf) WIN_INLINE {
    const int j0 = kt.at(n) * TILE;
    sv(vb + (long long)j0 * a.ldv, s.nk - 1 - j0, l0 + (2 + buf) * TB);
  };
  const int iw = i0 + wave * 32, i = iw + (lane & 31), ic = min(i, s.nq - 1);
  const int p = ic + off, hi = min(s.nk - 1, p + a.right), lo = p - a.left;
  const int wp0 = iw + off, wp1 = min(iw + 31, s.nq - 1) + off;
  const float c = a.scale * LOG2E;
  s16x8 qf[D / 16];
  load_cols<D>(qf, a.q + (long long)(s.q0 + ic) * a.ldq + pl.h * (D * 2));
  f32x16 o[D / 32], S0, S1;
  s16x8 P0[2], P1[2];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
  // probabilities are formed relative to a reference score m of the row, 2^(c s + neg), neg = -c m
  float neg = 0.f, l = 0.f;
  bool begun = false, all_begun = false;                               // the row has a reference; every row of the wave has
  auto scores = [&](const char* K, int u, f32x16& S) WIN_INLINE {
#pragma unroll
    for (int r = 0; r < 16; ++r) S[r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) S = mfma32<T>(row_frag32<D>(K, u * 32, ks), qf[ks], S);
  };
  auto values = [&](const char* V, int u, const s16x8 (&P)[2]) WIN_INLINE {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) o[dt] = mfma32<T>(col_frag32<D>(V, u * 32 + h * 16, dt), P[h], o[dt]);
  };
  auto row_max = [&](const f32x16& S) WIN_INLINE {
    float mx = S[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, S[r]);
    return both_halves(mx, true);
  };
  auto exponentials = [&](const f32x16& S, s16x8 (&P)[2]) WIN_INLINE {
    f32x16 E;
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      E[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[r], c, neg));
      t += E[r];
    }
    P[0] = pack8<T>(E, 0);
    P[1] = pack8<T>(E, 1);
    return t;
  };
  auto begin = [&](const f32x16& S) WIN_INLINE {
    const float mx = row_max(S);
    if (!begun && mx > -INFINITY) {
      neg = -mx * c;
      begun = true;
    }
    all_begun = __all(begun);
  };
  auto settle = [&](const f32x16& S, s16x8 (&P)[2], float t) WIN_INLINE {
    if (__any(t > 1024.f)) {
      const float to = fminf(neg, -row_max(S) * c);                    // (a row that sees nothing here: +inf, the minimum stays)
      float al = __builtin_amdgcn_exp2f(begun ? to - neg : 0.f);
      if (begun) neg = to;
      asm volatile("" : "+v"(al));                                     // (nothing of this before the branch)
      l *= al;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= al;
      t = exponentials(S, P);
    }
    l += t;
  };
  // One step = 32 keys: their exponentials (vector unit) beside the products of the 32 before (values) and after (scores), which do not
  // depend on them.  The scheduling groups deal the products out over the exponentials: one unit would wait for the other otherwise.
  // The reference is the maximum of the first keys a row sees, not a running one (a third of the vector work): it moves only when a sum
  // of 16 terms passes 2^10 - then the step's terms are formed again - and until then no term is over 2^10, which costs no precision.
  auto step = [&](int n, int u, const f32x16& S_, s16x8 (&P)[2], const char* V, const s16x8 (&Pv)[2], const char* K, f32x16& Sq) WIN_INLINE {
    f32x16 S = S_;
    s16x8 kf[D / 16], vf[2][D / 32];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) kf[ks] = row_frag32<D>(K, (1 - u) * 32, ks);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) vf[h][dt] = col_frag32<D>(V, (1 - u) * 32 + h * 16, dt);
    const int j0 = kt.at(n) * TILE + u * 32;
    const bool edge_hi = j0 + 31 > min(s.nk - 1, wp0 + a.right), edge_lo = j0 < wp1 - a.left;
    if (edge_lo | edge_hi) mask_keys(S, j0 + 4 * half, lo, hi, 0, edge_lo, edge_hi);
    if (!all_begun) begin(S);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < 16; ++r) Sq[r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      Sq = mfma32<T>(kf[ks], qf[ks], Sq);
      const int h = ks / (D / 32), dt = ks % (D / 32);
      o[dt] = mfma32<T>(vf[h][dt], Pv[h], o[dt]);
    }
    float t = exponentials(S, P);
    asm volatile("" : "+v"(P[0]), "+v"(P[1]), "+v"(t));                // formed here, not where they are next read
#pragma unroll
    for (int k = 0; k < D / 8; ++k) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);               // a matrix instruction
      __builtin_amdgcn_sched_group_barrier(0x002, 64 / (D / 8), 0);    // vector instructions
    }
    __builtin_amdgcn_sched_barrier(0);
    settle(S, P, t);
  };
  // K of tiles n, n + 1 and V of tiles n - 1, n are in use at tile n, so the next copies start between its two steps
  P1[0] = P1[1] = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
  if (kt.count) {
    stage_k(0, 0);
    stage_v(0, 0);
    stage_v(0, 1);                                                     // (what the first step multiplies by zeros has to be numbers)
  }
  tile_barrier();
  if (kt.count > 1) stage_k(1, 1);
  auto turn = [&](int n, int odd) WIN_INLINE {                                    // between a tile's two steps
    tile_barrier();
    if (n + 2 < kt.count) stage_k(n + 2, odd);
    if (n + 1 < kt.count) stage_v(n + 1, 1 - odd);
  };
  // (where tile n + 1 does not exist, its scores are formed from what stands there and not used)
  auto tile = [&](int n, int odd) WIN_INLINE {
    const char *K0 = lds + odd * TB, *K1 = lds + (1 - odd) * TB, *V0 = lds + (3 - odd) * TB, *V1 = lds + (2 + odd) * TB;
    step(n, 0, S0, P0, V0, P1, K0, S1);
    turn(n, odd);
    step(n, 1, S1, P1, V1, P0, K1, S0);
  };
  // The sinks' tiles, one after the other: often a few keys, of which a wave looks at the halves it sees.  (In the loop below, with
  // tiles between them and the window masked: 8191 tokens with four sinks 184 us instead of 180, others equal.)
  const int hw = iw < s.nq ? min(s.nk - 1, wp1 + a.right) : -1;
  auto seen = [&](int j0) WIN_INLINE { return j0 <= hw && (j0 < a.sinks || j0 + 31 >= wp0 - a.left); };
  auto alone = [&](f32x16& S, int j0, const char* V, int u) WIN_INLINE {
    mask_keys(S, j0 + 4 * half, lo, hi, a.sinks, true, true);
    if (!all_begun) begin(S);
    s16x8 P[2];
    const float t = exponentials(S, P);
    settle(S, P, t);
    values(V, u, P);
  };
  int n = 0;
  for (; n < kt.sink; ++n) {
    const int j0 = n * TILE, odd = n & 1;
    const bool seen0 = seen(j0), seen1 = seen(j0 + 32);
    if (seen0) scores(lds + odd * TB, 0, S0);
    if (seen1) scores(lds + odd * TB, 1, S1);
    turn(n, odd);
    if (seen0) alone(S0, j0, lds + (2 + odd) * TB, 0);
    if (seen1) alone(S1, j0 + 32, lds + (2 + odd) * TB, 1);
  }
  // the wave's own tiles of the window, na .. nb - 1 of the list.  The loop has no branch around the sums - where paths with and without
  // products meet, the compiler copies all of o - and two tiles a turn, so that all LDS addresses are constants.
  const int nb = hw < 0 ? 0 : hw / TILE - kt.first + kt.sink + 1;
  const int na = min(nb, kt.sink + max(0, max(0, wp0 - a.left) / TILE - kt.first));
  for (; n < na; ++n) turn(n, n & 1);
  if (n < nb) {
    scores(lds + (n & 1) * TB, 0, S0);
    if (n & 1) {
      tile(n, 1);
      ++n;
    }
    for (; n + 1 < nb; n += 2) {
      tile(n, 0);
      tile(n + 1, 1);
    }
    if (n < nb) {
      tile(n, 0);
      ++n;
    }
    values(lds + (2 + ((n - 1) & 1)) * TB, 1, P1);
  }
  for (; n < kt.count; ++n) turn(n, n & 1);
  if (i >= s.nq) return;
  l = both_halves(l, false);
  // 0: the row sees nothing (of a row that sees a key the reference's own term is 1); not a number: that is what out and lse say
  const float inv = l == 0.f ? 0.f : 1.f / l;
  char* po = a.out + (long long)(s.q0 + i) * a.ldo + pl.h * (D * 2);
  typedef __attribute__((ext_vector_type(4))) T T4;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      T4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (T)(o[dt][4 * g + e] * inv);
      *reinterpret_cast<T4*>(po + (dt * 32 + 8 * g + 4 * half) * 2) = y;
    }
  if (a.lse && half == 0) a.lse[(size_t)(s.q0 + i) * a.Hq + pl.h] = l == 0.f ? -INFINITY : (__log2f(l) - neg) * LN2;
}

// ---------------------------------------------------------------------------------------------- backward
// With P from the saved log-sum-exp and delta_i = sum_d dO_id O_id:
//     dV_j = sum_i P_ij dO_i     dS_ij = P_ij (dO_i . V_j - delta_i)     dQ_i = scale sum_j dS_ij K_j     dK_j = scale sum_i dS_ij Q_i
// Two kernels that form S and dO V^T again, one over queries (dQ), one over keys (dK, dV; the query heads that share a key head are
// summed in the workgroup): 7 products for the 5 of one kernel with atomic sums, but every sum has one fixed order.

// dQ and delta: the forward's walk, S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T.  Bound: as above, with three products
// for one exponential (matrix unit 44 % of the time, vector unit 53 %, LDS 22 %): the clips of above 142 us = 758 TFLOP/s, the packed texts
// 86 us = 480 (with the turn back, which takes 2 and 7 of these).  delta is formed from the forward's rounded out, half a step off at most,
// so that the forward need not leave 32-bit rows.
template <class T, int D>
__global__ __launch_bounds__(256, 2) void win_bwd_q_kernel(WinArgs a) {
  constexpr int TB = TILE * D * 2;
  __shared__ __attribute__((aligned(1024))) char lds[4 * TB];
  const int tiles = (a.max_q + 127) / 128;
  Place pl;
  if (!place(a, tiles, a.Hq, pl)) return;
  const Seq s = load_seq(a, pl.b);
  const int i0 = (tiles - 1 - pl.tile) * 128;
  if (i0 >= s.nq) {
    if (const int4 t = a.seqs[pl.b]; a.clear && left_out(a, t)) clear_rows<D>(a.dq, a.lddq, t.x, t.y, a.rows_q, pl.h, pl.tile, tiles);
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int off = s.nk - s.nq, hk = pl.h / (a.Hq / a.Hkv);
  const KeyTiles kt = key_tiles(a, s.nk, i0 + off, min(i0 + 127, s.nq - 1) + off);
  const char* kb = a.k + (long long)s.k0 * a.ldk + hk * (D * 2);
  const char* vb = a.v + (long long)s.k0 * a.ldv + hk * (D * 2);
  const uint32_t l0 = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) char*)lds);
  const Stager<D> sk(a.ldk), sv(a.ldv);
  auto stage = [&](int n, int buf) WIN_INLINE {
    const int j0 = kt.at(n) * TILE;
    sk(kb + (long long)j0 * a.ldk, s.nk - 1 - j0, l0 + buf * 2 * TB);
    sv(vb + (long long)j0 * a.ldv, s.nk - 1 - j0, l0 + buf * 2 * TB + TB);
  };
  const int iw = i0 + wave * 32, i = iw + (lane & 31), ic = min(i, s.nq - 1);
  const int p = ic + off, hi = min(s.nk - 1, p + a.right), lo = p - a.left;
  const int wp0 = iw + off, wp1 = min(iw + 31, s.nq - 1) + off;
  const float c = a.scale * LOG2E;
  const long long row = s.q0 + ic;
  s16x8 qf[D / 16], df[D / 16];
  load_cols<D>(qf, a.q + row * a.ldq + pl.h * (D * 2));
  load_cols<D>(df, a.dout + row * a.lddo + pl.h * (D * 2));
  float delta = 0.f;
  {
    s16x8 of[D / 16];
    load_cols<D>(of, a.o + row * a.ldo + pl.h * (D * 2));
    typedef __attribute__((ext_vector_type(8))) T T8;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const T8 x = __builtin_bit_cast(T8, df[ks]), y = __builtin_bit_cast(T8, of[ks]);
#pragma unroll
      for (int e = 0; e < 8; ++e) delta += (float)x[e] * (float)y[e];
    }
    delta = both_halves(delta, false);
  }
  float lse2 = a.lse[(size_t)row * a.Hq + pl.h] * LOG2E;
  if (lse2 == -INFINITY) lse2 = 0.f;                                   // a row that sees nothing: every pair of it is masked below
  if (i < s.nq && half == 0) {
    a.lse2[(size_t)pl.h * a.rows_q + row] = lse2;
    a.delta[(size_t)pl.h * a.rows_q + row] = delta;
  }
  f32x16 dq[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[dt][r] = 0.f;
  auto tile = [&](int n, int odd) WIN_INLINE {
    tile_barrier();
    if (n + 1 < kt.count) stage(n + 1, 1 - odd);
    const int j0 = kt.at(n) * TILE;
    if (iw >= s.nq || j0 > min(s.nk - 1, wp1 + a.right) || (j0 + TILE - 1 < wp0 - a.left && j0 >= a.sinks)) return;
    const char* Kt = lds + odd * 2 * TB;
    const char* Vt = Kt + TB;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int ju = j0 + u * 32;
      // 32 keys that no query of the wave sees.  Heads of 64 look at both halves of a tile together: without a branch between them the
      // compiler lays one half's products beside the other's exponentials (two 16-frame clips 139 us, with a branch 143; heads of 128,
      // where the registers do not allow that: six packed texts 82 us without this one, 79 with it)
      if (D == 128 && (ju > min(s.nk - 1, wp1 + a.right) || (ju + 31 < wp0 - a.left && ju >= a.sinks))) continue;
      f32x16 st, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) st[r] = dp[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        st = mfma32<T>(row_frag32<D>(Kt, u * 32, ks), qf[ks], st);
        dp = mfma32<T>(row_frag32<D>(Vt, u * 32, ks), df[ks], dp);
      }
      const bool edge_hi = ju + 31 > min(s.nk - 1, wp0 + a.right), edge_lo = ju < wp1 - a.left && ju + 31 >= a.sinks;
      if (edge_lo | edge_hi) mask_keys(st, ju + 4 * half, lo, hi, a.sinks, edge_lo, edge_hi);
#pragma unroll
      for (int r = 0; r < 16; ++r) st[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r], c, -lse2)) * (dp[r] - delta);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const s16x8 sf = pack8<T>(st, h);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) dq[dt] = mfma32<T>(col_frag32<D>(Kt, u * 32 + h * 16, dt), sf, dq[dt]);
      }
    }
  };
  if (kt.count) stage(0, 0);
  int n = 0;
  for (; n + 1 < kt.count; n += 2) {                                   // two tiles a turn: LDS addresses are constants
    tile(n, 0);
    tile(n + 1, 1);
  }
  if (n < kt.count) tile(n, 0);
  if (i >= s.nq) return;
  if (a.turns) turn_back<D>(dq, a.turns + row, a.rows_q);
  char* po = a.dq + row * a.lddq + pl.h * (D * 2);
  typedef __attribute__((ext_vector_type(4))) T T4;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      T4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (T)(dq[dt][4 * g + e] * a.scale);
      *reinterpret_cast<T4*>(po + (dt * 32 + 8 * g + 4 * half) * 2) = y;
    }
}

// a tile of 64 queries of head h, with their gradients, lse2 and delta, into the LDS
template <int D> OAT_DEV void stage_queries(const WinArgs& a, const Seq& s, const Stager<D>& sq, const Stager<D>& sd, int h, int t, uint32_t l, int wave) {
  const int i0 = t * TILE, last = s.nq - 1 - i0;
  const long long row = s.q0 + i0;
  sq(a.q + row * a.ldq + h * (D * 2), last, l);
  sd(a.dout + row * a.lddo + h * (D * 2), last, l + TILE * D * 2);
  if (wave < 2) {
    const float* src = (wave ? a.delta : a.lse2) + (size_t)h * a.rows_q + row;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
                 : : "v"((uint32_t)min((int)(threadIdx.x & 63), last) * 4u), "s"(src), "s"(__builtin_amdgcn_readfirstlane(l + 2 * TILE * D * 2 + wave * 256)) : "memory", "m0");
  }
}
// a slab: [dK, dV][D][32 keys]; slots of 32 sinks: (piece, half of its tiles), last the window's own
template <int D> OAT_DEV float* slab(const WinArgs& a, int b, int hk, int group, int slot, bool is_v) {
  return a.slabs + ((((size_t)(b * a.Hkv + hk) * a.groups + group) * (2 * a.pieces + 1) + slot) * 2 + is_v) * (D * 32);
}

// dK and dV: one launch of two kinds of workgroups.
//
// The sinks' keys are seen by every later query: the workgroup that owns them would walk the whole sequence while the others walk a
// window.  So the pairs beyond the window (the far ones) are taken by workgroups of their own (far_keys): 32 sink keys and one of
// `pieces` shares of the far queries each, where waves 0, 1 form dV and waves 2, 3 dK of the tile's two halves.  Those sums, and what
// the window gives the sinks, go to 32-bit slabs that win_bwd_sink_kernel adds in a fixed order.  The far workgroups are short and come
// last in the launch, where they fill its end: two clips of 7057 tokens 179 us for all of it, six packed texts 115; in a launch of their
// own 184 + 16 and 112 + 24, first in the launch 179 and 129.
template <class T, int D> OAT_DEV void far_keys(const WinArgs& a, char* lds, int block) {
  constexpr int TB = TILE * D * 2, ST = 2 * TB + 512;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, G = a.Hq / a.Hkv;
  const int piece = block % a.pieces, bhg = block / a.pieces, group = bhg % a.groups, hk = bhg / a.groups % a.Hkv, b = bhg / a.groups / a.Hkv;
  const Seq s = load_seq(a, b);
  const int j0 = group * 32;
  if (j0 >= s.nk || j0 >= a.sinks) return;
  const int off = s.nk - s.nq, j = j0 + (lane & 31), jc = min(j, s.nk - 1), jend = min(j0 + 31, s.nk - 1);
  // key j is seen from beyond its window by queries lo(j) .. the last
  auto lo = [&](int j) WIN_INLINE { return j + a.left - off + 1; };
  const int i0 = max(0, lo(j0)), t0 = i0 / TILE, nt = s.nq - 1 < i0 ? 0 : (s.nq - 1) / TILE - t0 + 1;
  const int na = __builtin_amdgcn_readfirstlane((int)((long long)nt * G * piece / a.pieces));
  const int nb = __builtin_amdgcn_readfirstlane((int)((long long)nt * G * (piece + 1) / a.pieces));
  const uint32_t l0 = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) char*)lds);
  const Stager<D> sq(a.ldq), sd(a.lddo);
  auto stage = [&](int n) WIN_INLINE { stage_queries<D>(a, s, sq, sd, hk * G + n / nt, t0 + n % nt, l0 + (n & 1) * ST, wave); };
  const float c = a.scale * LOG2E;
  s16x8 kf[D / 16], vf[D / 16];
  load_cols<D>(kf, a.k + (long long)(s.k0 + jc) * a.ldk + hk * (D * 2));
  load_cols<D>(vf, a.v + (long long)(s.k0 + jc) * a.ldv + hk * (D * 2));
  const int ilo = lo(j), ihi = j < min(s.nk, a.sinks) ? s.nq - 1 : -1;
  const bool do_k = wave >= 2, all_sinks = jend < a.sinks;
  const int u = wave & 1;
  f32x16 sum[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[dt][r] = 0.f;
  if (na < nb) stage(na);
  for (int n = na; n < nb; ++n) {
    tile_barrier();
    if (n + 1 < nb) stage(n + 1);
    const int iu = (t0 + n % nt) * TILE + u * 32;
    if (iu >= s.nq || iu + 31 < i0) continue;
    const char* Qt = lds + (n & 1) * ST;
    const char* Dt = Qt + TB;
    const float* Lt = reinterpret_cast<const float*>(Dt + TB) + u * 32 + 4 * half;
    f32x16 st;
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) st = mfma32<T>(row_frag32<D>(Qt, u * 32, ks), kf[ks], st);
    if (iu < lo(jend) || iu + 31 >= s.nq || !all_sinks) mask_queries(st, iu + 4 * half, ilo, ihi);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 ls = *reinterpret_cast<const f32x4*>(Lt + 8 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) st[4 * g + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[4 * g + e], c, -ls[e]));
    }
    if (do_k) {
      f32x16 dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) dp = mfma32<T>(row_frag32<D>(Dt, u * 32, ks), vf[ks], dp);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 de = *reinterpret_cast<const f32x4*>(Lt + 64 + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) st[4 * g + e] *= dp[4 * g + e] - de[e];
      }
    }
    const char* Xt = do_k ? Qt : Dt;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const s16x8 f = pack8<T>(st, h);
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) sum[dt] = mfma32<T>(col_frag32<D>(Xt, u * 32 + h * 16, dt), f, sum[dt]);
    }
  }
  float* sl = slab<D>(a, b, hk, group, 2 * piece + u, !do_k) + (lane & 31);
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) sl[(dt * 32 + 8 * (r >> 2) + 4 * half + (r & 3)) * 32] = sum[dt][r];
}

template <int D> OAT_DEV void clear_keys(const WinArgs& a, const Place& pl, int tiles) {
  const int4 t = a.seqs[pl.b];
  if (!left_out(a, t)) return;
  clear_rows<D>(a.dk, a.lddk, t.z, t.w, a.rows_k, pl.h, pl.tile, tiles);
  clear_rows<D>(a.dv, a.lddv, t.z, t.w, a.rows_k, pl.h, pl.tile, tiles);
}

// 128 keys, 32 a wave: S = Q K^T, dP = dO V^T with the key as the column, dV^T += dO^T P, dK^T += Q^T dS; queries and their gradients
// pass through the LDS in tiles of 64, with their lse2 and delta.  Bound: as above (four products for one exponential; matrix unit
// 43 % of the time, vector unit 48 %, LDS 33 %): the clips of above 182 us = 788 TFLOP/s.
template <class T, int D> OAT_DEV void window_keys(const WinArgs& a, char* lds) {
  constexpr int TB = TILE * D * 2, ST = 2 * TB + 512;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, G = a.Hq / a.Hkv;
  Place pl;
  const int tiles = (a.max_k + 127) / 128;
  if (!place(a, tiles, a.Hkv, pl)) return;
  const Seq s = load_seq(a, pl.b);
  const int j0 = pl.tile * 128;
  if (j0 >= s.nk) {
    if (a.clear) clear_keys<D>(a, pl, tiles);
    return;
  }
  const int off = s.nk - s.nq;
  const bool split = a.groups > 0;                                     // the sinks' far queries are other workgroups' (far_keys)
  // the queries that see key j: i = lo(j) .. hi(j)
  auto lo = [&](int j) WIN_INLINE { return j - a.right - off; };
  auto hi = [&](int j) WIN_INLINE { return !split && j < a.sinks ? s.nq - 1 : min(s.nq - 1, j + a.left - off); };
  const int jend = min(j0 + 127, s.nk - 1);
  const int i0 = max(0, lo(j0)), i1 = !split && j0 < a.sinks ? s.nq - 1 : hi(jend);
  const int t0 = i0 / TILE, nt = i1 < i0 ? 0 : i1 / TILE - t0 + 1, count = nt * G;
  const uint32_t l0 = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) char*)lds);
  const Stager<D> sq(a.ldq), sd(a.lddo);
  auto stage = [&](int n) WIN_INLINE { stage_queries<D>(a, s, sq, sd, pl.h * G + n / nt, t0 + n % nt, l0 + (n & 1) * ST, wave); };
  const int jw = j0 + wave * 32, j = jw + (lane & 31), jc = min(j, s.nk - 1), jwe = min(jw + 31, s.nk - 1);
  const float c = a.scale * LOG2E;
  s16x8 kf[D / 16], vf[D / 16];
  load_cols<D>(kf, a.k + (long long)(s.k0 + jc) * a.ldk + pl.h * (D * 2));
  load_cols<D>(vf, a.v + (long long)(s.k0 + jc) * a.ldv + pl.h * (D * 2));
  const int ilo = lo(j), ihi = j < s.nk ? hi(j) : -1;
  const bool sink_w = !split && jwe < a.sinks;                                    // the wave's keys are sinks all
  // queries wlo .. whi see a key of the wave, flo .. fhi see them all
  const int wlo = lo(jw), whi = !split && jw < a.sinks ? s.nq - 1 : hi(jwe);
  const int flo = lo(jwe), fhi = sink_w ? s.nq - 1 : min(s.nq - 1, jw + a.left - off);
  f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[dt][r] = dv[dt][r] = 0.f;
  if (count) stage(0);
  for (int n = 0; n < count; ++n) {
    tile_barrier();
    if (n + 1 < count) stage(n + 1);
    const int it = (t0 + n % nt) * TILE;
    const char* Qt = lds + (n & 1) * ST;
    const char* Dt = Qt + TB;
    const float* Lt = reinterpret_cast<const float*>(Dt + TB);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int iu = it + u * 32;
      if (jw >= s.nk || iu > whi || iu + 31 < wlo) continue;
      f32x16 st, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) st[r] = dp[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) st = mfma32<T>(row_frag32<D>(Qt, u * 32, ks), kf[ks], st);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) dp = mfma32<T>(row_frag32<D>(Dt, u * 32, ks), vf[ks], dp);
      if (iu < flo || iu + 31 > fhi) mask_queries(st, iu + 4 * half, ilo, ihi);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 ls = *reinterpret_cast<const f32x4*>(Lt + u * 32 + 8 * g + 4 * half);
        const f32x4 de = *reinterpret_cast<const f32x4*>(Lt + 64 + u * 32 + 8 * g + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          st[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r], c, -ls[e]));
          dp[r] -= de[e];
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const s16x8 pf = pack8<T>(st, h);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) dv[dt] = mfma32<T>(col_frag32<D>(Dt, u * 32 + h * 16, dt), pf, dv[dt]);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] *= st[r];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const s16x8 sf = pack8<T>(dp, h);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) dk[dt] = mfma32<T>(col_frag32<D>(Qt, u * 32 + h * 16, dt), sf, dk[dt]);
      }
    }
  }
  if (split && jw < a.sinks) {
    float* sk = slab<D>(a, pl.b, pl.h, jw / 32, 2 * a.pieces, false) + (lane & 31);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int d = dt * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
        sk[d * 32] = dk[dt][r];
        sk[(D + d) * 32] = dv[dt][r];
      }
    return;
  }
  if (j >= s.nk) return;
  if (a.turns) turn_back<D>(dk, a.turns + s.k0 + j, a.rows_q);
  char* pk = a.dk + (long long)(s.k0 + j) * a.lddk + pl.h * (D * 2);
  char* pv = a.dv + (long long)(s.k0 + j) * a.lddv + pl.h * (D * 2);
  typedef __attribute__((ext_vector_type(4))) T T4;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      T4 x, y;
#pragma unroll
      for (int e = 0; e < 4; ++e) { x[e] = (T)(dk[dt][4 * g + e] * a.scale); y[e] = (T)dv[dt][4 * g + e]; }
      *reinterpret_cast<T4*>(pk + (dt * 32 + 8 * g + 4 * half) * 2) = x;
      *reinterpret_cast<T4*>(pv + (dt * 32 + 8 * g + 4 * half) * 2) = y;
    }
}

// The same for 64 keys, heads of 128: two waves share 32 keys.  Each forms P and dS of one half of a tile, hands one of them to the other
// through the LDS, and then one adds up dV, the other dK, of the whole tile: every product is formed once, and a wave holds one sum
// instead of two (64 instead of 128 registers at D = 128), so that two waves fit a SIMD.  The packed texts of above, with the sinks' far
// queries and the turn back: 113 us = 488 TFLOP/s (matrix unit 29 %, vector unit 24 %, 1.4 waves on a SIMD).
template <class T, int D> OAT_DEV void window_keys_in_pairs(const WinArgs& a, char* lds) {
  constexpr int TB = TILE * D * 2, ST = 2 * TB + 512;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, G = a.Hq / a.Hkv;
  Place pl;
  const int tiles = (a.max_k + 63) / 64;
  if (!place(a, tiles, a.Hkv, pl)) return;
  const Seq s = load_seq(a, pl.b);
  const int j0 = pl.tile * 64;
  if (j0 >= s.nk) {
    if (a.clear) clear_keys<D>(a, pl, tiles);
    return;
  }
  const int off = s.nk - s.nq;
  const bool split = a.groups > 0;                                     // the sinks' far queries are other workgroups' (far_keys)
  auto lo = [&](int j) WIN_INLINE { return j - a.right - off; };       // the queries that see key j
  auto hi = [&](int j) WIN_INLINE { return !split && j < a.sinks ? s.nq - 1 : min(s.nq - 1, j + a.left - off); };
  const int jend = min(j0 + 63, s.nk - 1);
  const int i0 = max(0, lo(j0)), i1 = !split && j0 < a.sinks ? s.nq - 1 : hi(jend);
  const int t0 = i0 / TILE, nt = i1 < i0 ? 0 : i1 / TILE - t0 + 1, count = nt * G;
  const uint32_t l0 = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) char*)lds);
  const Stager<D> sq(a.ldq), sd(a.lddo);
  auto stage = [&](int g, int t, int buf) WIN_INLINE { stage_queries<D>(a, s, sq, sd, pl.h * G + g, t, l0 + buf * ST, wave); };
  const int u = wave >> 1;                                             // the wave's half of a tile; 0 adds up dV, 1 dK
  const int jw = j0 + (wave & 1) * 32, j = jw + (lane & 31), jc = min(j, s.nk - 1), jwe = min(jw + 31, s.nk - 1);
  const float c = a.scale * LOG2E;
  s16x8 kf[D / 16], vf[D / 16];
  load_cols<D>(kf, a.k + (long long)(s.k0 + jc) * a.ldk + pl.h * (D * 2));
  load_cols<D>(vf, a.v + (long long)(s.k0 + jc) * a.ldv + pl.h * (D * 2));
  const int ilo = lo(j), ihi = j < s.nk ? hi(j) : -1;
  const bool sink_w = !split && jwe < a.sinks;                         // the wave's keys are sinks all
  // queries wlo .. whi see a key of the wave, flo .. fhi see them all
  const int wlo = lo(jw), whi = !split && jw < a.sinks ? s.nq - 1 : hi(jwe);
  const int flo = lo(jwe), fhi = sink_w ? s.nq - 1 : min(s.nq - 1, jw + a.left - off);
  f32x16 sum[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[dt][r] = 0.f;
  char* const mine = lds + 2 * ST + wave * 2048 + lane * 16;
  const char* const other = lds + 2 * ST + (wave ^ 2) * 2048 + lane * 16;
  int g1 = 0, t1 = t0;                                                 // head and tile that is staged next
  if (count) {
    stage(0, t0, 0);
    t1 = t0 + 1;
  }
  int t = t0;
  for (int n = 0; n < count; ++n) {
    tile_barrier();
    if (t1 == t0 + nt) { t1 = t0; ++g1; }
    if (n + 1 < count) stage(g1, t1, (n + 1) & 1);
    const int iu = t * TILE + u * 32;
    const char* Qt = lds + (n & 1) * ST;
    const char* Dt = Qt + TB;
    const float* Lt = reinterpret_cast<const float*>(Dt + TB) + u * 32 + 4 * half;
    s16x8 keep[2];
    if (jw >= s.nk || iu > whi || iu + 31 < wlo) {
      keep[0] = keep[1] = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
      *reinterpret_cast<s16x8*>(mine) = keep[0];
      *reinterpret_cast<s16x8*>(mine + 1024) = keep[0];
    } else {
      f32x16 st, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) st[r] = dp[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        st = mfma32<T>(row_frag32<D>(Qt, u * 32, ks), kf[ks], st);
        dp = mfma32<T>(row_frag32<D>(Dt, u * 32, ks), vf[ks], dp);
      }
      if (iu < flo || iu + 31 > fhi) mask_queries(st, iu + 4 * half, ilo, ihi);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 ls = *reinterpret_cast<const f32x4*>(Lt + 8 * g), de = *reinterpret_cast<const f32x4*>(Lt + 64 + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          st[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r], c, -ls[e]));
          dp[r] -= de[e];
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] *= st[r];
      const s16x8 p0 = pack8<T>(st, 0), p1 = pack8<T>(st, 1), s0 = pack8<T>(dp, 0), s1 = pack8<T>(dp, 1);
      *reinterpret_cast<s16x8*>(mine) = u ? p0 : s0;
      *reinterpret_cast<s16x8*>(mine + 1024) = u ? p1 : s1;
      keep[0] = u ? s0 : p0;
      keep[1] = u ? s1 : p1;
    }
    const char* Xt = u ? Qt : Dt;
    auto add = [&](const s16x8 (&x)[2], int half_of_tile) WIN_INLINE {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) sum[dt] = mfma32<T>(col_frag32<D>(Xt, half_of_tile * 32 + h * 16, dt), x[h], sum[dt]);
    };
    add(keep, u);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const s16x8 got[2] = {*reinterpret_cast<const s16x8*>(other), *reinterpret_cast<const s16x8*>(other + 1024)};
    add(got, 1 - u);
    if (++t == t0 + nt) t = t0;
    ++t1;
  }
  if (split && jw < a.sinks) {
    float* sl = slab<D>(a, pl.b, pl.h, jw / 32, 2 * a.pieces, !u) + (lane & 31);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) sl[(dt * 32 + 8 * (r >> 2) + 4 * half + (r & 3)) * 32] = sum[dt][r];
    return;
  }
  if (j >= s.nk) return;
  if (u && a.turns) turn_back<D>(sum, a.turns + s.k0 + j, a.rows_q);
  const float f = u ? a.scale : 1.f;
  char* po = (u ? a.dk + (long long)(s.k0 + j) * a.lddk : a.dv + (long long)(s.k0 + j) * a.lddv) + pl.h * (D * 2);
  typedef __attribute__((ext_vector_type(4))) T T4;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      T4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (T)(sum[dt][4 * g + e] * f);
      *reinterpret_cast<T4*>(po + (dt * 32 + 8 * g + 4 * half) * 2) = x;
    }
}

// heads of 64: both sums of 32 keys fit a wave beside another wave's (two 16-frame clips 180 us, shared in pairs 194); heads of 128:
// they do not (six packed texts 182 us, in pairs 138)
constexpr int keys_of_a_workgroup(int D) { return D == 64 ? 128 : 64; }
template <class T, int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void win_bwd_kv_kernel(WinArgs a) {
  constexpr int ST = 2 * TILE * D * 2 + 512;
  __shared__ __attribute__((aligned(1024))) char lds[2 * ST + (D == 64 ? 0 : 8192)];
  const int far = (int)blockIdx.x - (int)gridDim.x + a.far_blocks;
  if (far >= 0) far_keys<T, D>(a, lds, far);
  else if constexpr (D == 64) window_keys<T, D>(a, lds);
  else window_keys_in_pairs<T, D>(a, lds);
}

// the sinks' slabs, added slot by slot (every eighth one a thread, then the eight): a workgroup = 32 keys, two chunks of 8 values of dK or
// dV half a head apart, which are pairs of the rotary positions
template <class T, int D>
__global__ __launch_bounds__(256) void win_bwd_sink_kernel(WinArgs a) {
  __shared__ float part[8][16][32];
  const int key = threadIdx.x & 31, w = threadIdx.x >> 5;
  const bool is_v = blockIdx.y >= D / 16;
  const int d8 = blockIdx.y % (D / 16) * 8;
  const int group = blockIdx.x % a.groups, h = blockIdx.x / a.groups % a.Hkv, b = blockIdx.x / a.groups / a.Hkv;
  const Seq s = load_seq(a, b);
  if (group * 32 >= min(a.sinks, s.nk)) return;
  const int slots = 2 * a.pieces + 1;
  const float* sl = slab<D>(a, b, h, group, w, is_v) + d8 * 32 + key;
  float x[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = 0.f;
#pragma unroll 2
  for (int i = w; i < slots; i += 8, sl += 8 * 2 * D * 32) {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] += sl[(e < 8 ? e : e - 8 + D / 2) * 32];
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) part[w][e][key] = x[e];
  __syncthreads();
  const int j = group * 32 + key;
  if (w || j >= s.nk) return;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
#pragma unroll
    for (int k = 1; k < 8; ++k) x[e] += part[k][e][key];
  }
  const long long row = s.k0 + j;
  if (!is_v && a.turns) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 t = a.turns[(size_t)(d8 + e) * a.rows_q + row], y = rope_turn(x[e], x[8 + e], float2{t.x, -t.y});
      x[e] = y.x;
      x[8 + e] = y.y;
    }
  }
  typedef __attribute__((ext_vector_type(8))) T T8;
  char* p = (is_v ? a.dv + row * a.lddv : a.dk + row * a.lddk) + h * (D * 2);
  const float f = is_v ? 1.f : a.scale;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    T8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (T)(x[8 * c + e] * f);
    *reinterpret_cast<T8*>(p + (d8 + c * (D / 2)) * 2) = y;
  }
}

// how the far pairs of the sinks are split: groups of 32 sink keys, pieces of their queries, each about half as many as a window's tile walks
// (as many: packed texts 121 us instead of 115); 0 groups: the sinks' own tiles walk all queries.  That takes max_q / 64 steps where a window's tile takes (left + right + 128) / 64:
// split where it is over 512 queries longer.  (Of many sinks - over 512 keys - the tiles themselves are enough workgroups, and the slabs
// would be large.)
struct FarSplit { int groups, pieces; };
static FarSplit far_split(int B, int Hq, int Hkv, int D, int max_q, int max_k, int left, int sinks) {
  const long long rows = min((long long)max_q, (long long)max_k - left);
  if (sinks < 1 || min(sinks, max_k) > 512 || rows <= 512 || B < 1) return {0, 0};
  const int groups = (min(sinks, max_k) + 31) / 32;
  const long long pieces = min(256ll, 2 * rows / (left + 128) + 1);
  if ((long long)B * Hkv * groups * max(pieces, (long long)D / 8) >= 1ll << 23) return {0, 0};  // (a launch holds 2^32 threads)
  return {groups, (int)pieces};
}
static size_t slab_floats(const FarSplit& f, int B, int Hkv, int D) {
  return (size_t)B * Hkv * f.groups * (2 * f.pieces + 1) * 2 * D * 32;
}

static bool rows_wrong(const void* p, long long ld, int heads, int D) {
  return !p || (uintptr_t)p % 16 || ld % 8 || ld < (long long)heads * D || ld > (1 << 22);
}
static int window_wrong(const char* what, const void* seqs, int B, int max_q, int max_k, int rows_q, int rows_k, int Hq, int Hkv, int D,
                        int dtype, int sinks, float scale) {
  const char* w = nullptr;
  if (D != 64 && D != 128) w = "heads of 64 or 128 values";
  else if (dtype != 0 && dtype != 1) w = "element type: 0 (bf16) or 1 (fp16)";
  else if (Hkv < 1 || Hq < 1 || Hq % Hkv) w = "the query heads are not a multiple of the key heads";
  else if (B < 0 || max_q < 0 || max_k < 0 || rows_q < 0 || rows_k < 0 || max_q > (1 << 29) || max_k > (1 << 29)) w = "lengths of 0 to 2^29";
  else if (B && !seqs) w = "the table of sequences is missing";
  else if ((uintptr_t)seqs % 16) w = "the table of sequences is not aligned to 16 bytes";
  else if (sinks < 0 || sinks > (1 << 29)) w = "sinks of 0 to 2^29";
  else if (!(scale > 0.f && scale < 1e30f)) w = "the scale is not a positive number";
  else if ((long long)B * Hq * (max_q / 128 + 1) >= (1ll << 22) || (long long)B * Hkv * (max_k / 64 + 1) >= (1ll << 22)) w = "more than 2^22 tiles";
  if (!w) return 0;
  char msg[160];
  snprintf(msg, sizeof msg, "%s: %s", what, w);
  set_error(msg);
  return -2;
}
static int far(int n) { return n < 0 || n > (1 << 29) ? 1 << 29 : n; }      // a window without that edge

}  // namespace oat

using namespace oat;

#define WIN_FWD(T, D) win_fwd_kernel<T, D>
#define WIN_Q(T, D) win_bwd_q_kernel<T, D>
#define WIN_KV(T, D) win_bwd_kv_kernel<T, D>
#define WIN_SINK(T, D) win_bwd_sink_kernel<T, D>
#define WIN_LAUNCH(kernel, grid) WIN_LAUNCH2(kernel, dim3(grid))
#define WIN_LAUNCH2(kernel, grid)                                                                                    \
  do {                                                                                                               \
    const dim3 g_ = (grid);                                                                                          \
    if (dtype == 0 && D == 64) OAT_LAUNCH((kernel(bf16, 64)), g_, dim3(256), 0, s, a);                                 \
    else if (dtype == 0) OAT_LAUNCH((kernel(bf16, 128)), g_, dim3(256), 0, s, a);                                      \
    else if (D == 64) OAT_LAUNCH((kernel(_Float16, 64)), g_, dim3(256), 0, s, a);                                      \
    else OAT_LAUNCH((kernel(_Float16, 128)), g_, dim3(256), 0, s, a);                                                  \
  } while (0)

int oat::attn_window_fwd(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, void* out, long long ldo,
                         float* lse, const int* seqs, int B, int max_q, int max_k, int rows_q, int rows_k, int Hq, int Hkv, int D, int dtype,
                         int left, int right, int sinks, float scale, int clear, void* stream) {
  if (int rc = window_wrong("attn_window_fwd", seqs, B, max_q, max_k, rows_q, rows_k, Hq, Hkv, D, dtype, sinks, scale)) return rc;
  if (B == 0 || max_q == 0 || rows_q == 0) return 0;
  if (rows_wrong(q, ldq, Hq, D) || rows_wrong(out, ldo, Hq, D) || (rows_k && (rows_wrong(k, ldk, Hkv, D) || rows_wrong(v, ldv, Hkv, D)))) {
    set_error("attn_window_fwd: q, k, v, out need 16-byte aligned rows (pitch a multiple of 8, at least the heads, at most 2^22 values)");
    return -2;
  }
  WinArgs a{};
  a.q = (const char*)q; a.k = (const char*)k; a.v = (const char*)v; a.out = (char*)out; a.lse = lse;
  a.ldq = ldq * 2; a.ldk = ldk * 2; a.ldv = ldv * 2; a.ldo = ldo * 2;
  a.seqs = (const int4*)seqs;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.left = far(left); a.right = far(right); a.sinks = sinks;
  a.max_q = max_q; a.max_k = max_k; a.rows_q = rows_q; a.rows_k = rows_k; a.scale = scale; a.clear = clear;
  hipStream_t s = (hipStream_t)stream;
  const int tiles = (max_q + 127) / 128;
  a.run = deal_run(B, Hq, Hq / Hkv, tiles, rows_q, max_q);
  WIN_LAUNCH(WIN_FWD, deal_grid((long long)B * Hq * tiles, a.run));
  return check_launch("attn_window_fwd");
}

extern "C" int oat_attn_window_fwd(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, void* out,
                                   long long ldo, float* lse, const int* seqs, int B, int max_q, int max_k, int rows_q, int rows_k,
                                   int Hq, int Hkv, int D, int dtype, int left, int right, int sinks, float scale, void* stream) {
  return attn_window_fwd(q, ldq, k, ldk, v, ldv, out, ldo, lse, seqs, B, max_q, max_k, rows_q, rows_k, Hq, Hkv, D, dtype, left, right, sinks,
                         scale, 0, stream);
}

extern "C" size_t oat_attn_window_bwd_workspace_bytes(int rows_q, int B, int max_q, int max_k, int Hq, int Hkv, int D, int left, int sinks) {
  if (rows_q < 0 || Hq < 1 || Hkv < 1 || D < 1) return 0;
  return ((size_t)rows_q * Hq * 2 + slab_floats(far_split(B, Hq, Hkv, D, max_q, max_k, far(left), sinks), B, Hkv, D)) * 4;
}

int oat::attn_window_bwd(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, const void* out,
                         long long ldo, const float* lse, const void* dout, long long lddo, void* dq, long long lddq, void* dk,
                         long long lddk, void* dv, long long lddv, const int* seqs, int B, int max_q, int max_k, int rows_q, int rows_k,
                         int Hq, int Hkv, int D, int dtype, int left, int right, int sinks, float scale, void* workspace,
                         size_t workspace_bytes, const float2* turns, int clear, void* stream) {
  if (int rc = window_wrong("attn_window_bwd", seqs, B, max_q, max_k, rows_q, rows_k, Hq, Hkv, D, dtype, sinks, scale)) return rc;
  if (B == 0) return 0;
  if (rows_q && (rows_wrong(q, ldq, Hq, D) || rows_wrong(out, ldo, Hq, D) || rows_wrong(dout, lddo, Hq, D) || rows_wrong(dq, lddq, Hq, D) || !lse)) {
    set_error("attn_window_bwd: q, out, dout, dq need 16-byte aligned rows (pitch a multiple of 8, at least the heads, at most 2^22 values), and lse");
    return -2;
  }
  if (rows_k && (rows_wrong(k, ldk, Hkv, D) || rows_wrong(v, ldv, Hkv, D) || rows_wrong(dk, lddk, Hkv, D) || rows_wrong(dv, lddv, Hkv, D))) {
    set_error("attn_window_bwd: k, v, dk, dv need 16-byte aligned rows (pitch a multiple of 8, at least the heads, at most 2^22 values)");
    return -2;
  }
  if (rows_q && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < oat_attn_window_bwd_workspace_bytes(rows_q, B, max_q, max_k, Hq, Hkv, D, left, sinks))) { set_error("attn_window_bwd: the workspace is too small, or not aligned to 16 bytes"); return -3; }
  WinArgs a{};
  a.q = (const char*)q; a.k = (const char*)k; a.v = (const char*)v; a.o = (const char*)out; a.dout = (const char*)dout;
  a.lse = const_cast<float*>(lse); a.dq = (char*)dq; a.dk = (char*)dk; a.dv = (char*)dv;
  a.ldq = ldq * 2; a.ldk = ldk * 2; a.ldv = ldv * 2; a.ldo = ldo * 2; a.lddo = lddo * 2; a.lddq = lddq * 2; a.lddk = lddk * 2; a.lddv = lddv * 2;
  a.lse2 = (float*)workspace; a.delta = a.lse2 + (size_t)rows_q * Hq;
  a.seqs = (const int4*)seqs;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.left = far(left); a.right = far(right); a.sinks = sinks;
  a.max_q = max_q; a.max_k = max_k; a.rows_q = rows_q; a.rows_k = rows_k; a.scale = scale; a.clear = clear;
  a.turns = turns;
  hipStream_t s = (hipStream_t)stream;
  if (max_q && rows_q) {
    const int tiles = (max_q + 127) / 128;
    a.run = deal_run(B, Hq, Hq / Hkv, tiles, rows_q, max_q);
    WIN_LAUNCH(WIN_Q, deal_grid((long long)B * Hq * tiles, a.run));
  }
  const FarSplit f = rows_q ? far_split(B, Hq, Hkv, D, max_q, max_k, a.left, sinks) : FarSplit{0, 0};
  a.groups = f.groups;
  a.pieces = f.pieces;
  a.slabs = a.delta + (size_t)rows_q * Hq;
  if (max_k && rows_k) {
    const int tiles = (max_k + keys_of_a_workgroup(D) - 1) / keys_of_a_workgroup(D);
    a.run = deal_run(B, Hkv, 1, tiles, rows_k, max_k);
    a.far_blocks = B * Hkv * f.groups * f.pieces;
    WIN_LAUNCH(WIN_KV, deal_grid((long long)B * Hkv * tiles, a.run) + a.far_blocks);
  }
  if (max_k && rows_k && f.groups) WIN_LAUNCH2(WIN_SINK, dim3(B * Hkv * f.groups, D / 8));
  return check_launch("attn_window_bwd");
}

extern "C" int oat_attn_window_bwd(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, const void* out,
                                   long long ldo, const float* lse, const void* dout, long long lddo, void* dq, long long lddq, void* dk,
                                   long long lddk, void* dv, long long lddv, const int* seqs, int B, int max_q, int max_k, int rows_q,
                                   int rows_k, int Hq, int Hkv, int D, int dtype, int left, int right, int sinks, float scale,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  return attn_window_bwd(q, ldq, k, ldk, v, ldv, out, ldo, lse, dout, lddo, dq, lddq, dk, lddk, dv, lddv, seqs, B, max_q, max_k, rows_q, rows_k,
                         Hq, Hkv, D, dtype, left, right, sinks, scale, workspace, workspace_bytes, nullptr, 0, stream);
}
