// Tiles, fragments and visibility shared by the windowed-attention kernels (attn_window.hip: forward and backward).
//
// Matrix instruction 32x32x16 (16-bit operands, fp32 sums):
//   A: lane l holds A[row = l & 31][k = (l >> 5) * 8 .. +8]     B: lane l holds B[k = (l >> 5) * 8 .. +8][col = l & 31]
//   C: lane l, register r holds C[row = 8 * (r >> 2) + 4 * (l >> 5) + (r & 3)][col = l & 31]
// A product's C can be the next product's B without leaving the registers, because the order of a sum's terms is free: registers
// 8c .. 8c + 7 of a lane are the rows 16 c + 8 * (e >> 2) + 4 * (l >> 5) + (e & 3), e = 0..7, and the A fragments of that next
// product are read from the LDS (transposing reads) in the same order of k.
#pragma once
#include "rope.h"
#include <stdio.h>

namespace oat {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

#define WIN_INLINE __attribute__((always_inline))

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

template <class T> OAT_DEV f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c);
template <> OAT_DEV f32x16 mfma32<bf16>(s16x8 a, s16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> OAT_DEV f32x16 mfma32<_Float16>(s16x8 a, s16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// registers 8c .. 8c + 7 as a B fragment: one rounding of each value to the operands' type (the matrix unit takes no 32-bit operand
// at this rate); the sums stay in 32 bits
template <class T> OAT_DEV s16x8 pack8(const f32x16& x, int c) {
  typedef __attribute__((ext_vector_type(8))) T T8;
  T8 y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = (T)x[8 * c + e];
  return __builtin_bit_cast(s16x8, y);
}

// ---- tiles of 64 rows in the LDS, rows of D 16-bit values in chunks of 16 bytes.  Chunk c of row r stands at place c ^ swz(r): a row
// fragment (16 rows, one chunk) and a transposing read (4 rows of 4 neighbouring chunks, or 8 of 2) then touch every bank alike.
template <int D> OAT_DEV int swz(int r) { return (D == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2) | ((r >> 2) & 1) << 1 | ((r >> 3) & 1); }

constexpr int TILE = 64;

// Asynchronous copies of tiles by 256 threads: rows 0 .. TILE - 1 from `base` (wave-uniform), pitch `ldb` bytes.  A whole tile takes one
// lane offset for all of its pieces (a piece is 256 / CPR rows, and swz repeats with them): no vector instructions.  In a ragged tile the
// rows past `last` repeat that row, so that no memory outside the sequence is read and nothing but its own finite values stands there.
template <int D> struct Stager {
  static constexpr int CPR = D / 8, RPP = 256 / CPR;                   // chunks of a row, rows of a piece
  uint32_t ldb, off, wave;
  OAT_DEV Stager(long long ld) {
    const int tid = threadIdx.x, r = tid / CPR;
    ldb = (uint32_t)ld;
    off = r * ldb + (((tid % CPR) ^ swz<D>(r)) << 4);
    wave = __builtin_amdgcn_readfirstlane(tid >> 6) * 1024;
  }
  OAT_DEV void operator()(const char* base, int last, uint32_t lds) const {
    lds += wave;
    if (last >= TILE - 1) {
#pragma unroll
      for (int i = 0; i < TILE / RPP; ++i) glds16(base + (size_t)i * RPP * ldb, off, lds + i * 4096);
    } else {
      const int tid = threadIdx.x, r0 = tid / CPR;
      const uint32_t ch = ((tid % CPR) ^ swz<D>(r0)) << 4;
#pragma unroll
      for (int i = 0; i < TILE / RPP; ++i) glds16(base, (uint32_t)min(i * RPP + r0, last) * ldb + ch, lds + i * 4096);
    }
  }
  OAT_DEV static void glds16(const char* base, uint32_t lane_off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(lane_off), "s"(base), "s"(lds) : "memory", "m0");
  }
};
// A fragment: rows rb .. rb + 31 of a tile, k = 16 ks .. +16
template <int D> OAT_DEV s16x8 row_frag32(const char* tile, int rb, int ks) {
  const int lane = threadIdx.x & 63, r = lane & 31;
  return *reinterpret_cast<const s16x8*>(tile + (rb + r) * (D * 2) + (((2 * ks + (lane >> 5)) ^ swz<D>(r)) << 4));
}
// A fragment of the transposed tile: rows d = 32 dt .. +32, k = the tile's rows kb .. kb + 15 in the order of a C fragment's registers
template <int D> OAT_DEV s16x8 col_frag32(const char* tile, int kb, int dt) {
  const int lane = threadIdx.x & 63, j = (lane >> 2) & 3, q4 = lane & 3;
  const int ch = dt * 4 + ((lane >> 4) & 1) * 2 + (q4 >> 1);
  s16x8 out;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = 8 * e + 4 * (lane >> 5) + j;
    const s16x4 h = lds_tr16(tile + (kb + r) * (D * 2) + ((ch ^ swz<D>(r)) << 4) + (q4 & 1) * 8);
#pragma unroll
    for (int x = 0; x < 4; ++x) out[4 * e + x] = h[x];
  }
  return out;
}
// B fragments of 32 rows in memory (row = the lane's column of the product)
template <int D> OAT_DEV void load_cols(s16x8 (&f)[D / 16], const char* row) {
  const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) f[ks] = *reinterpret_cast<const s16x8*>(row + (2 * ks + half) * 16);
}
// turns the sums of a row (C fragments of the transposed product: a lane holds half of one row) back by its pairs' cos and sin.  A pair is
// (d, d + D / 2): one register of two fragments.  `turns` points to the row's first pair, `pitch` rows a pair: the lanes read neighbouring
// rows (with the pairs of a row side by side a wave's read touched 64 lines: six packed texts' query gradients 80 -> 91 us; so: 87).
template <int D> OAT_DEV void turn_back(f32x16 (&x)[D / 32], const float2* turns, int pitch) {
  const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int dt = 0; dt < D / 64; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float2 w = turns[(size_t)(dt * 32 + 8 * (r >> 2) + 4 * half + (r & 3)) * pitch];
      const float2 y = rope_turn(x[dt][r], x[dt + D / 64][r], float2{w.x, -w.y});
      x[dt][r] = y.x;
      x[dt + D / 64][r] = y.y;
    }
}
// maximum / sum of a value over lanes l and l ^ 32 (one register swap of the halves, no LDS)
OAT_DEV float both_halves(float v, bool max) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
  const float x = __builtin_bit_cast(float, (int)r[0]), y = __builtin_bit_cast(float, (int)r[1]);
  return max ? fmaxf(x, y) : x + y;
}
// every wave's copies have landed and every wave is done reading what the next copies overwrite.  The compiler does not know of the
// copies, so the wait for them is asm; the builtin (vmcnt 0, lgkmcnt 0) after it tells the compiler that its own earlier loads are done:
// it would put waits for these into the loop, and those would wait for the next tile's copies too.
OAT_DEV void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x70);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ---- sequences and visibility.  Query i of a sequence stands at position p = i + nk - nq (its last query at its last key); it sees
// key j if  j <= p + right  and  (j >= p - left  or  j < sinks).
struct WinArgs {
  const char *q, *k, *v, *o, *dout;
  char *out, *dq, *dk, *dv;
  float* lse;                           // [rows_q, Hq], natural logarithm; -inf: the row sees nothing
  float *lse2, *delta;                  // backward: [Hq, rows_q], base 2; sum of dout * out
  long long ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;      // bytes
  const int4* seqs;                     // first query row, queries, first key row, keys
  float* slabs;                         // backward: the sinks' sums (win_bwd_kv_kernel)
  int B, Hq, Hkv, left, right, sinks, max_q, max_k, rows_q, rows_k;
  int run;                              // tiles that go to one XCD together
  int groups, pieces, far_blocks;       // how the sinks' far queries are split; their workgroups in the launch
  float scale;
  int clear;                            // rows of a sequence that is left out for its length get zeros (the layer's on packed rows do)
  const float2* turns;                  // backward: cos and sin of [D / 2, rows_q] pairs (p, p + D / 2) to turn dq and dk back by, or null
};
struct Seq { int q0, nq, k0, nk; };
// a sequence that does not fit the buffers (or the launch) is taken as empty, by the attention and by the caches: nothing outside is read or
// written
OAT_DEV bool rows_fit(int first, int n, int most, int rows) { return first >= 0 && n >= 0 && n <= most && (long long)first + n <= rows; }
OAT_DEV bool left_out(const WinArgs& a, const int4& s) { return !(rows_fit(s.x, s.y, a.max_q, a.rows_q) && rows_fit(s.z, s.w, a.max_k, a.rows_k)); }
OAT_DEV Seq load_seq(const WinArgs& a, int b) {
  const int4 s = a.seqs[b];
  return left_out(a, s) ? Seq{0, 0, 0, 0} : Seq{s.x, s.y, s.z, s.w};
}
// Zeros for head h's rows of a sequence that load_seq left out though its rows lie in the buffer (there are more than stated, or its other
// side does not fit), for buffers in which every row is one sequence's: no other workgroup writes them.  `part` of `parts` workgroups.
template <int D> OAT_DEV void clear_rows(char* base, long long ld, int first, int n, int rows, int h, int part, int parts) {
  if (!rows_fit(first, n, n, rows)) return;
  constexpr int CPR = D / 8;
  for (long long t = part * 256 + (int)threadIdx.x; t < (long long)n * CPR; t += parts * 256)
    *reinterpret_cast<f32x4*>(base + (first + t / CPR) * ld + h * (D * 2) + t % CPR * 16) = f32x4{0.f, 0.f, 0.f, 0.f};
}
// blockIdx -> (tile, head, sequence).  Workgroups go to the 8 XCDs in turn; the (sequence, head, tile) list is dealt to the XCDs in runs of
// a.run tiles, which share keys in one L2 (deal_run below).
struct Place { int b, h, tile; };
OAT_DEV bool place(const WinArgs& a, int tiles, int heads, Place& p) {
  const int k = blockIdx.x >> 3, c = k / a.run, i = (c * 8 + (blockIdx.x & 7)) * a.run + k - c * a.run;
  if (i >= tiles * heads * a.B) return false;
  const int bh = i / tiles;
  p.tile = i - bh * tiles;
  p.b = bh / heads;
  p.h = bh - p.b * heads;
  return true;
}
// The length of a run.  In a batch of different lengths short runs of an odd length, so that every XCD gets some of each sequence and of
// its empty places (six packed texts, from one contiguous share an XCD: forward 83 -> 65 us, dQ 105 -> 84, dK and dV 137 -> 107; whole
// heads: 64, 82, 130).  Else whole key heads with the query heads that share them, or single heads, where they come out even, or an
// eighth of the list.
inline int deal_run(int B, int heads, int group, int tiles, long long rows, int longest) {
  const long long units = (long long)B * heads;
  if (rows * 10 < 9ll * B * longest) return 5;
  auto even = [](long long u) { return u % 8 == 0 || u >= 64; };
  if (even(units / group)) return tiles * group;
  return even(units) ? tiles : (int)((units * tiles + 7) / 8);
}
inline unsigned deal_grid(long long n, int run) { return (unsigned)((n + 8ll * run - 1) / (8ll * run) * (8ll * run)); }

// The visibility of the pair that register r of a C fragment holds, with the fixed side (a query's keys lo .. hi and sinks, or a key's
// queries) folded into bounds on the register's row number: row <= hi and (row >= lo or row < sink), no branches.
struct Bounds {
  int lo, hi, sink;
  OAT_DEV bool sees(int r) const {
    const int row = 8 * (r >> 2) + (r & 3);
    return (row <= hi) & ((row >= lo) | (row < sink));
  }
};
// masks the scores of 32 keys (the first at jb for this lane's half; lo .. hi and the sinks are what its query sees).  Most tiles that
// are not seen whole lie across one edge only: one comparison each.  (The empty asm keeps the comparisons behind the caller's branch.)
OAT_DEV void mask_keys(f32x16& S, int jb, int lo, int hi, int sinks, bool edge_lo, bool edge_hi) {
  asm volatile("" : "+v"(jb));
  const Bounds bd{lo - jb, hi - jb, sinks - jb};
  if (!edge_lo) {
#pragma unroll
    for (int r = 0; r < 16; ++r) S[r] = 8 * (r >> 2) + (r & 3) <= bd.hi ? S[r] : -INFINITY;
  } else if (!edge_hi && sinks <= __builtin_amdgcn_readfirstlane(jb)) {
#pragma unroll
    for (int r = 0; r < 16; ++r) S[r] = 8 * (r >> 2) + (r & 3) >= bd.lo ? S[r] : -INFINITY;
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) S[r] = bd.sees(r) ? S[r] : -INFINITY;
  }
}
// and of 32 queries, ilo .. ihi being those that see this lane's key
OAT_DEV void mask_queries(f32x16& S, int ib, int ilo, int ihi) {
  asm volatile("" : "+v"(ib));
  const int lo = ilo - ib, hi = ihi - ib;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = 8 * (r >> 2) + (r & 3);
    S[r] = (row >= lo) & (row <= hi) ? S[r] : -INFINITY;
  }
}
// the key tiles (of 64) that queries at positions p0 .. p1 see: those of the sinks, then those of the window
struct KeyTiles {
  int sink, first, count;
  OAT_DEV int at(int n) const { return n < sink ? n : first + n - sink; }
};
OAT_DEV KeyTiles key_tiles(const WinArgs& a, int nk, int p0, int p1) {
  const int hi = min(nk - 1, p1 + a.right);
  if (hi < 0) return {0, 0, 0};
  const int end = hi / TILE + 1;
  const int sink = min((min(a.sinks, nk) + TILE - 1) / TILE, end);
  const int first = max(max(0, p0 - a.left) / TILE, sink);
  return {sink, first, sink + max(0, end - first)};
}

// oat_attn_window_fwd and _bwd; clear: WinArgs::clear; `turns` (may be null): dq and dk are turned back by these before they are rounded
// (WinArgs::turns; rows_q = rows_k)
int attn_window_fwd(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, void* out, long long ldo,
                    float* lse, const int* seqs, int B, int max_q, int max_k, int rows_q, int rows_k, int Hq, int Hkv, int D, int dtype,
                    int left, int right, int sinks, float scale, int clear, void* stream);
int attn_window_bwd(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, const void* out, long long ldo,
                    const float* lse, const void* dout, long long lddo, void* dq, long long lddq, void* dk, long long lddk, void* dv,
                    long long lddv, const int* seqs, int B, int max_q, int max_k, int rows_q, int rows_k, int Hq, int Hkv, int D, int dtype,
                    int left, int right, int sinks, float scale, void* workspace, size_t workspace_bytes, const float2* turns, int clear, void* stream);

}  // namespace oat
