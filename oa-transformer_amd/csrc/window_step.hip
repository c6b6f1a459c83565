// The serving form of windowed attention: one new token of every sequence against a cache of keys and values, and the copy of a
// prompt's keys and values into such a cache.
//
// A cache holds `cap` slots per sequence.  Plain: token t stands in slot t.  Rolling: the first `sinks` tokens stay, the others go
// round in the remaining slots, slot(t) = sinks + (t - sinks) mod (cap - sinks), so a window of cap - sinks tokens and the sinks is
// all that is ever held.  The order of a softmax's terms is free, so the step never unrolls a rolling cache.
#include "attn_window.h"

namespace oat {

template <class T> OAT_DEV f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c);
template <> OAT_DEV f32x4 mfma16<bf16>(s16x8 a, s16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> OAT_DEV f32x4 mfma16<_Float16>(s16x8 a, s16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

struct StepArgs {
  const char* qkv; long long ldqkv;                  // bytes; q heads | k heads | v heads
  const int* past;                                   // [B] tokens before this one
  const int* pos;                                    // [B, n_axes]
  char *kc, *vc;
  long long kb, ks, kh, vb, vs, vh;                  // cache strides in bytes: sequence, slot, head
  char* out; long long ldo;
  float *pieces, *sums; int* tickets;                // [B, Hq, splits, D], [B, Hq, splits, 2] (maximum in base 2, sum), [B, Hkv]
  int B, Hq, Hkv, cap, left, sinks, rolling, splits, turn;
  float scale;
  OatRope rope;
};

// the pieces' sums pass between workgroups of different XCDs: agent-scope accesses go past the L2s that are not shared, so that no
// fence has to write back and drop whole caches (with __threadfence a workgroup took 100 us instead of 10)
OAT_DEV void put(float* p, float v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
OAT_DEV void put2(float* p, f32x2 v) {
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), __builtin_bit_cast(unsigned long long, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
OAT_DEV f32x2 get2(const float* p) {
  return __builtin_bit_cast(f32x2, __hip_atomic_load(reinterpret_cast<const unsigned long long*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

constexpr int SK = 32;                               // keys of a wave's tile
template <int D> constexpr int step_lds() { return 4 * 2 * SK * D * 2; }

// One workgroup = one piece of the visible keys of one (sequence, key head), for up to 16 of the query heads that share it; a wave
// takes every fourth tile of 32 keys.  Bound: the cache is read once - HBM; so keys and values go straight to the LDS (asynchronous, no
// register waits on them), a wave waits for its own tiles only, and while it works on a tile's keys its values are on their way (and the
// next keys while it works on these): 64 KB in flight per CU, with 64 KB of LDS a workgroup (D = 128), so that two or more share a CU.  S^T = K Q^T and
// O^T += V^T P^T on 16x16x32 products with the query head as the column: shared heads cost nothing more than one.
// The new token's query and key are turned here (one angle per pair and workgroup); the workgroup of the piece that holds the
// new token writes its row to the cache first.  The turned query and key and the probabilities are rounded to the operands' 16 bits (the
// cache holds no more, the matrix unit takes no more); scores, statistics and sums are 32-bit.  Pieces are joined by the workgroup that
// finishes last, in a fixed order.
// Measured: 64 sequences of up to 4096 tokens, 32 / 8 heads of 128: 576 MB in 117 us = 4.9 TB/s; two of 65536 visible tokens: 537 MB in
// 107 us = 5.0 (a large copy: 4.9 to 5.4); one of 512, 12 heads of 64: 7.8 us, a chain of dependent loads.
template <class T, int D>
__global__ __launch_bounds__(256, 2) void win_step_kernel(StepArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  __shared__ __attribute__((aligned(16))) T qs[16 * D];
  __shared__ float2 cs[64];
  __shared__ float wm[4][16], wl[4][16];
  __shared__ int last;
  constexpr int CPR = D / 8, NI = SK * CPR / 64, TB = SK * D * 2;
  const int G = a.Hq / a.Hkv, gts = (G + 15) / 16;
  const int piece = blockIdx.x % a.splits, rest = blockIdx.x / a.splits;
  const int gt = rest % gts, hk = rest / gts % a.Hkv, b = rest / gts / a.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g0 = gt * 16, ng = min(16, G - g0);
  const int p = a.past[b];
  if (p < 0 || (!a.rolling && p >= a.cap)) {         // a sequence that takes no part (or has no slot left): zeros, the cache stays
    if (piece == 0)
      for (int t = tid; t < ng * D; t += 256) reinterpret_cast<T*>(a.out + b * a.ldo)[(hk * G + g0) * D + t] = (T)0.f;
    return;
  }
  const int all = p < 0x7fffffff ? p + 1 : p;
  const int nv = a.rolling ? min(all, a.cap) : (a.left < all - 1 - a.sinks ? a.sinks + a.left + 1 : all);
  const int shift = a.rolling ? 0 : all - nv;
  const int chunk = ((nv + a.splits - 1) / a.splits + 4 * SK - 1) / (4 * SK) * (4 * SK);
  const int parts = (nv + chunk - 1) / chunk, ta = piece * chunk, tb = min(nv, ta + chunk);
  if (ta >= nv) return;
  const char* row = a.qkv + b * a.ldqkv;
  const int np = a.turn ? a.rope.n_pairs : 0;
  auto turned = [&](const T* x, int d) {             // value d of a head, turned
    if (d >= 2 * np) return (float)x[d];
    const int pr = a.rope.interleaved ? d >> 1 : d < np ? d : d - np;
    const bool second = a.rope.interleaved ? d & 1 : d >= np;
    const int iu = a.rope.interleaved ? 2 * pr : pr, iv = a.rope.interleaved ? 2 * pr + 1 : pr + np;
    const float u = (float)x[iu], v = (float)x[iv];
    const float2 y = rope_turn(u, v, cs[pr]);
    return second ? y.y : y.x;
  };
  if (tid < np) cs[tid] = rope_cos_sin(a.pos[(size_t)b * a.rope.n_axes + a.rope.axis[tid]], a.rope.turns[tid], false);
  __syncthreads();
  char* kb = a.kc + b * a.kb + hk * a.kh;
  char* vb = a.vc + b * a.vb + hk * a.vh;
  const int slot = !a.rolling || p < a.sinks ? p : a.sinks + (p - a.sinks) % (a.cap - a.sinks);
  const int mark = a.rolling ? slot : nv - 1;        // where the new token stands among the visible ones
  if (mark >= ta && mark < tb) {
    if (tid < D) {
      reinterpret_cast<T*>(kb + slot * a.ks)[tid] = (T)turned(reinterpret_cast<const T*>(row) + (a.Hq + hk) * D, tid);
      reinterpret_cast<T*>(vb + slot * a.vs)[tid] = reinterpret_cast<const T*>(row)[(a.Hq + a.Hkv + hk) * D + tid];
    }
  }
  for (int t = tid; t < 16 * D; t += 256) {
    const int g = t / D, d = t % D;
    qs[t] = g < ng ? (T)turned(reinterpret_cast<const T*>(row) + (hk * G + g0 + g) * D, d) : (T)0.f;
  }
  tile_barrier();                                    // the new row has been written before any wave reads it
  const uint32_t l0 = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) char*)lds) + wave * 2 * TB;
  const char *Kt = lds + wave * 2 * TB, *Vt = Kt + TB;
  auto stage = [&](const char* base, long long pitch, int t0, uint32_t dst) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = i * 64 + lane, r = c / CPR, ch = (c % CPR) ^ swz<D>(r);
      const int t = min(t0 + r, tb - 1);
      const long long slot = t < a.sinks ? t : t + shift;
      asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                   : : "v"(base + slot * pitch + ch * 16), "s"(dst + i * 1024) : "memory", "m0");
    }
  };
  auto landed = [] {                                 // all but the NI copies issued last
    if constexpr (NI == 8) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
  };
  const int gq = lane >> 4, r16 = lane & 15;
  const float c = a.scale * LOG2E;
  f32x4 o[D / 16];
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  int t0 = ta + wave * SK;
  if (t0 < tb) {
    stage(kb, a.ks, t0, l0);
    stage(vb, a.vs, t0, l0 + TB);
  }
  for (; t0 < tb; t0 += 4 * SK) {
    const bool more = t0 + 4 * SK < tb;
    landed();                                        // this tile's keys; its values are on their way
    f32x4 st[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      st[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) {
        const s16x8 kf = *reinterpret_cast<const s16x8*>(Kt + (u * 16 + r16) * (D * 2) + (((4 * ks + gq) ^ swz<D>(r16)) << 4));
        const s16x8 qf = *reinterpret_cast<const s16x8*>(qs + r16 * D + ks * 32 + gq * 8);
        st[u] = mfma16<T>(kf, qf, st[u]);
      }
    }
    if (t0 + SK > tb) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (t0 + u * 16 + 4 * gq + r >= tb) st[u][r] = -INFINITY;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (more) stage(kb, a.ks, t0 + 4 * SK, l0);      // the next keys take the place of these
    float mx = m;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, st[u][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float al = __builtin_amdgcn_exp2f((m - mx) * c);            // mx is finite: a tile holds one visible key at least
    m = mx;
    l *= al;
    typedef __attribute__((ext_vector_type(8))) T T8;
    T8 pf;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = __builtin_amdgcn_exp2f((st[u][r] - mx) * c);
        l += e;
        pf[4 * u + r] = (T)e;
      }
    if (more) landed();                              // this tile's values
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const int j = (lane >> 2) & 3, q4 = lane & 3;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      s16x8 vf;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 4 * gq + j;
        const s16x4 h = lds_tr16(Vt + (16 * e + r) * (D * 2) + (((2 * dt + (q4 >> 1)) ^ swz<D>(r)) << 4) + (q4 & 1) * 8);
#pragma unroll
        for (int x = 0; x < 4; ++x) vf[4 * e + x] = h[x];
      }
      o[dt] *= al;
      o[dt] = mfma16<T>(vf, __builtin_bit_cast(s16x8, pf), o[dt]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (more) stage(vb, a.vs, t0 + 4 * SK, l0 + TB);
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  // the four waves' sums meet in the LDS: [wave][head][D]
  __syncthreads();
  float* os = reinterpret_cast<float*>(lds);
  if (gq == 0) { wm[wave][r16] = m; wl[wave][r16] = l; }
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) *reinterpret_cast<f32x4*>(os + (wave * 16 + r16) * D + dt * 16 + 4 * gq) = o[dt];
  __syncthreads();
  for (int t = tid; t < ng * D; t += 256) {
    const int g = t / D, d = t % D;
    float mm = wm[0][g];
#pragma unroll
    for (int w = 1; w < 4; ++w) mm = fmaxf(mm, wm[w][g]);
    float ll = 0.f, oo = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float e = __builtin_amdgcn_exp2f((wm[w][g] - mm) * c);
      ll += wl[w][g] * e;
      oo += os[(w * 16 + g) * D + d] * e;
    }
    const int h = hk * G + g0 + g;
    if (parts == 1) {
      reinterpret_cast<T*>(a.out + b * a.ldo)[h * D + d] = (T)(oo / ll);
    } else {
      const size_t at = (size_t)(b * a.Hq + h) * a.splits + piece;
      put(a.pieces + at * D + d, oo);
      if (d == 0) put2(a.sums + at * 2, f32x2{mm * c, ll});
    }
  }
  if (parts == 1) return;
  tile_barrier();                                    // this workgroup's sums are where every XCD sees them
  if (tid == 0) {
    int* tk = a.tickets + b * a.Hkv + hk;
    last = __hip_atomic_fetch_add(tk, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts * gts - 1;
    if (last) __hip_atomic_store(tk, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  // join: the weight of every piece of four heads into the LDS, then each team of D / 2 lanes adds every TEAMS-th piece (eight bytes a
  // lane, four pieces of four heads in flight), and the teams' sums meet in the LDS
  constexpr int TEAMS = 512 / D;
  float* wt = reinterpret_cast<float*>(lds);                           // [4][256]
  f32x2* red = reinterpret_cast<f32x2*>(lds + 4096);                   // [TEAMS][4][D / 2]
  const int team = tid / (D / 2), dl = tid % (D / 2);
  for (int gb = 0; gb < G; gb += 4) {
    const size_t row0 = (size_t)(b * a.Hq + hk * G + gb) * a.splits;
    __syncthreads();
    {
      // a wave = one head: maximum, sum and weights of its pieces, up to 256
      f32x2 ml[4];
      float mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = k * 64 + lane;
        ml[k] = i < parts && gb + wave < G ? get2(a.sums + (row0 + (size_t)wave * a.splits + i) * 2) : f32x2{-INFINITY, 0.f};
        mm = fmaxf(mm, ml[k][0]);
      }
      mm = wave_max(mm);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        ml[k][0] = ml[k][0] > -INFINITY ? __builtin_amdgcn_exp2f(ml[k][0] - mm) : 0.f;
        ll += ml[k][0] * ml[k][1];
      }
      ll = wave_sum(ll);
#pragma unroll
      for (int k = 0; k < 4; ++k) wt[wave * 256 + k * 64 + lane] = gb + wave < G ? ml[k][0] / ll : 0.f;
    }
    __syncthreads();
    f32x2 acc[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) acc[g] = f32x2{0.f, 0.f};
    for (int i = team; i < parts; i += 4 * TEAMS) {
      f32x2 x[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int g = 0; g < 4; ++g)                                    // (past the last piece or head: the last one, with weight 0)
          x[k][g] = get2(a.pieces + (row0 + (size_t)min(g, G - 1 - gb) * a.splits + min(i + k * TEAMS, parts - 1)) * D + 2 * dl);
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int g = 0; g < 4; ++g) acc[g] += (i + k * TEAMS < parts ? wt[g * 256 + i + k * TEAMS] : 0.f) * x[k][g];
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) red[(team * 4 + g) * (D / 2) + dl] = acc[g];
    __syncthreads();
    for (int t = tid; t < min(4, G - gb) * (D / 2); t += 256) {
      f32x2 v = red[t];
      for (int w = 1; w < TEAMS; ++w) v += red[w * 4 * (D / 2) + t];
      T* po = reinterpret_cast<T*>(a.out + b * a.ldo) + (hk * G + gb) * D + 2 * t;
      po[0] = (T)v[0];
      po[1] = (T)v[1];
    }
  }
}

// ---- a prompt's keys and values into a cache: slot by slot, the token that holds it at the end (no two writers of a slot)
struct FillArgs {
  const char *k, *v;
  long long ldk, ldv;
  char *kc, *vc;
  long long kb, ks, kh, vb, vs, vh;
  const int4* seqs;
  int B, Hkv, cap, sinks, rows_k, max_k, chunks;     // chunks: 16-byte pieces of a head
  int rows_q, max_q;                                 // the attention's, where the prompt's queries have to fit too; max_q < 0: they need not
};
__global__ __launch_bounds__(256) void cache_fill_kernel(FillArgs a) {
  const int b = blockIdx.y, per = a.Hkv * a.chunks;
  const int4 s = a.seqs[b];
  if (!rows_fit(s.z, s.w, a.max_k, a.rows_k) || (a.max_q >= 0 && !rows_fit(s.x, s.y, a.max_q, a.rows_q))) return;
  const int S = min(a.sinks, a.cap), W = a.cap - S;
  const long long total = (long long)min(a.cap, s.w) * per;
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < total; t += (long long)gridDim.x * 256) {
    const int slot = (int)(t / per), c = (int)(t - (long long)slot * per), h = c / a.chunks, x = c - h * a.chunks;
    const int tok = slot < S ? slot : slot + (s.w - 1 - slot) / W * W;
    const long long row = s.z + tok;
    *reinterpret_cast<f32x4*>(a.kc + b * a.kb + slot * a.ks + h * a.kh + x * 16) = *reinterpret_cast<const f32x4*>(a.k + row * a.ldk + c * 16);
    *reinterpret_cast<f32x4*>(a.vc + b * a.vb + slot * a.vs + h * a.vh + x * 16) = *reinterpret_cast<const f32x4*>(a.v + row * a.ldv + c * 16);
  }
}

static int fail(const char* what, const char* why) {
  char msg[192];
  snprintf(msg, sizeof msg, "%s: %s", what, why);
  set_error(msg);
  return -2;
}
// whether two of the places {a sequence's, a slot's, a head's} of a cache overlap: by rising stride, each dimension has to step over all of
// the smaller ones (a dimension of one takes no steps)
static bool places_share(const long long* st, int B, int cap, int Hkv, int D) {
  const int n[3] = {B, cap, Hkv};
  long long extent = D;
  bool done[3] = {n[0] <= 1, n[1] <= 1, n[2] <= 1};
  for (int k = 0; k < 3; ++k) {
    int least = -1;
    for (int i = 0; i < 3; ++i)
      if (!done[i] && (least < 0 || st[i] < st[least])) least = i;
    if (least < 0) return false;
    if (st[least] < extent) return true;
    extent += st[least] * (n[least] - 1);
    done[least] = true;
  }
  return false;
}
static const char* cache_wrong(const void* k, const void* v, const long long* st, int B, int cap, int Hkv, int D, int sinks) {
  if (D != 64 && D != 128) return "heads of 64 or 128 values";
  if (B < 0 || Hkv < 1 || cap < 1 || cap > (1 << 29) || sinks < 0 || sinks > (1 << 29)) return "no key heads, or a cache of no slots (or more than 2^29)";
  if (!k || !v || !st) return "the cache is missing";
  if (((uintptr_t)k | (uintptr_t)v) % 16) return "the cache is not aligned to 16 bytes";
  for (int i = 0; i < 6; ++i)
    if (st[i] < 0 || st[i] % 8) return "the cache's strides are not multiples of 8 values";
  return nullptr;
}
// pieces a cache may be split into: about four workgroups per CU in all
static int most_pieces(int B, int Hkv) { return min(256, 1 + 1024 / max(1, B * Hkv)); }

}  // namespace oat

using namespace oat;

extern "C" size_t oat_attn_window_step_workspace_bytes(int B, int Hq, int Hkv, int D) {
  if (B < 1 || Hq < 1 || Hkv < 1) return 0;
  return ((size_t)B * Hq * most_pieces(B, Hkv) * (D + 2) + (size_t)B * Hkv) * 4;
}

extern "C" int oat_attn_window_step(const void* qkv, long long ldqkv, const int* past, void* kc, void* vc, const long long* strides, int cap,
                                    void* out, long long ldo, int B, int Hq, int Hkv, int D, int dtype, int left, int sinks, int rolling,
                                    float scale, const OatRope* rope, const int* pos, void* workspace, size_t workspace_bytes, void* stream) {
  const char* me = "attn_window_step";
  if (B == 0) return 0;
  if (const char* w = cache_wrong(kc, vc, strides, B, cap, Hkv, D, sinks)) return fail(me, w);
  if (dtype != 0 && dtype != 1) return fail(me, "element type: 0 (bf16) or 1 (fp16)");
  if (Hq < 1 || Hq % Hkv) return fail(me, "the query heads are not a multiple of the key heads");
  if (places_share(strides, B, cap, Hkv, D) || places_share(strides + 3, B, cap, Hkv, D)) return fail(me, "slots of the cache share memory");
  if (!(scale > 0.f && scale < 1e30f)) return fail(me, "the scale is not a positive number");
  if (!qkv || !out || !past) return fail(me, "qkv, out and the counts of past tokens are needed");
  if (((uintptr_t)qkv | (uintptr_t)out) % 16 || ldqkv % 8 || ldo % 8 || ldqkv < (long long)(Hq + 2 * Hkv) * D || ldo < (long long)Hq * D)
    return fail(me, "qkv and out need 16-byte aligned rows of all their heads");
  if (rolling && (sinks >= cap || (left >= 0 && left != cap - sinks - 1))) return fail(me, "a rolling cache has sinks + left + 1 slots");
  if (rope) {
    if (const char* w = rope_wrong(rope, D)) return fail(me, w);
    if (!pos) return fail(me, "positions are needed to turn by");
  }
  // (of other sizes its tickets would stand elsewhere, where this call's may find sums instead of zeros)
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes != oat_attn_window_step_workspace_bytes(B, Hq, Hkv, D))
    return fail(me, "the workspace is not one of these sizes (B, Hq, Hkv, D), or not aligned to 16 bytes");
  if ((long long)B * Hkv * ((Hq / Hkv + 15) / 16) * most_pieces(B, Hkv) >= (1ll << 23)) return fail(me, "more than 2^23 pieces");
  StepArgs a{};
  a.qkv = (const char*)qkv; a.ldqkv = ldqkv * 2; a.past = past; a.pos = pos;
  a.kc = (char*)kc; a.vc = (char*)vc;
  a.kb = strides[0] * 2; a.ks = strides[1] * 2; a.kh = strides[2] * 2; a.vb = strides[3] * 2; a.vs = strides[4] * 2; a.vh = strides[5] * 2;
  a.out = (char*)out; a.ldo = ldo * 2;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.cap = cap; a.sinks = sinks; a.rolling = rolling != 0;
  a.left = left < 0 || left > (1 << 29) ? 1 << 29 : left;
  const long long seen = rolling ? cap : min((long long)cap, (long long)sinks + a.left + 1);
  // a piece of 512 keys is four tiles a wave; joining two pieces costs about what these take (12 heads, 512 keys: 7.6 us whole, 8.6 us in two)
  a.splits = (int)max(1ll, min((long long)most_pieces(B, Hkv), (seen + 511) / 512));
  a.turn = rope != nullptr;
  if (rope) a.rope = *rope;
  a.scale = scale;
  a.pieces = (float*)workspace;
  a.sums = a.pieces + (size_t)B * Hq * most_pieces(B, Hkv) * D;
  a.tickets = (int*)(a.sums + (size_t)B * Hq * most_pieces(B, Hkv) * 2);
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)(B * Hkv * ((Hq / Hkv + 15) / 16) * a.splits));
#define STEP_LAUNCH(T, DD)                                                       \
  do {                                                                           \
    OAT_MAX_LDS((win_step_kernel<T, DD>), step_lds<DD>());                        \
    OAT_LAUNCH(win_step_kernel<T, DD>, grid, dim3(256), step_lds<DD>(), s, a);    \
  } while (0)
  if (dtype == 0 && D == 64) STEP_LAUNCH(bf16, 64);
  else if (dtype == 0) STEP_LAUNCH(bf16, 128);
  else if (D == 64) STEP_LAUNCH(_Float16, 64);
  else STEP_LAUNCH(_Float16, 128);
#undef STEP_LAUNCH
  return check_launch(me);
}

static int cache_fill(const void* k, long long ldk, const void* v, long long ldv, const int* seqs, int B, int rows_k, int max_k, int rows_q,
                      int max_q, void* kc, void* vc, const long long* strides, int cap, int Hkv, int D, int sinks, void* stream) {
  const char* me = "window_cache_fill";
  if (B == 0) return 0;
  if (const char* w = cache_wrong(kc, vc, strides, B, cap, Hkv, D, sinks)) return fail(me, w);
  if (places_share(strides, B, cap, Hkv, D) || places_share(strides + 3, B, cap, Hkv, D)) return fail(me, "slots of the cache share memory");
  if (rows_k < 0 || max_k < 0 || B > 65535) return fail(me, "no rows, or more than 65535 sequences");
  if (rows_k == 0 || max_k == 0) return 0;
  if (!k || !v || !seqs || ((uintptr_t)k | (uintptr_t)v | (uintptr_t)seqs) % 16 || ldk % 8 || ldv % 8 || ldk < (long long)Hkv * D || ldv < (long long)Hkv * D)
    return fail(me, "k, v need 16-byte aligned rows of all key heads, and the table of sequences 16 bytes");
  FillArgs a{};
  a.k = (const char*)k; a.v = (const char*)v; a.ldk = ldk * 2; a.ldv = ldv * 2; a.kc = (char*)kc; a.vc = (char*)vc;
  a.kb = strides[0] * 2; a.ks = strides[1] * 2; a.kh = strides[2] * 2; a.vb = strides[3] * 2; a.vs = strides[4] * 2; a.vh = strides[5] * 2;
  a.seqs = (const int4*)seqs;
  a.B = B; a.Hkv = Hkv; a.cap = cap; a.sinks = sinks; a.rows_k = rows_k; a.max_k = max_k; a.chunks = D / 8;
  a.rows_q = rows_q; a.max_q = max_q;
  const long long n = (long long)min(cap, max_k) * Hkv * a.chunks;
  OAT_LAUNCH(cache_fill_kernel, dim3((unsigned)min((n + 255) / 256, 4096ll), B), dim3(256), 0, (hipStream_t)stream, a);
  return check_launch(me);
}

extern "C" int oat_window_cache_fill(const void* k, long long ldk, const void* v, long long ldv, const int* seqs, int B, int rows_k,
                                     int max_k, void* kc, void* vc, const long long* strides, int cap, int Hkv, int D, int sinks,
                                     void* stream) {
  return cache_fill(k, ldk, v, ldv, seqs, B, rows_k, max_k, 0, -1, kc, vc, strides, cap, Hkv, D, sinks, stream);
}

// ---- the counts of tokens that belong to a cache: those of a prompt, by the rule that the attention and the fill go by, and a step's, by
// the rule that the step goes by (in a launch of its own: a step's workgroups read the counts as long as any of them runs)
static __global__ __launch_bounds__(256) void cache_counts_kernel(int* past, const int4* seqs, int B, int rows, int longest) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b >= B) return;
  const int4 s = seqs[b];
  past[b] = rows_fit(s.x, s.y, longest, rows) && rows_fit(s.z, s.w, longest, rows) ? s.w : 0;
}

extern "C" int oat_window_cache_counts(int* past, const int* seqs, int B, int rows, int longest, void* stream) {
  const char* me = "window_cache_counts";
  if (B < 0 || rows < 0 || longest < 0) return fail(me, "a negative number of sequences, rows or tokens");
  if (B == 0) return 0;
  if (!past || !seqs || (uintptr_t)seqs % 16) return fail(me, "the counts, or the table of sequences (on 16 bytes), are missing");
  OAT_LAUNCH(cache_counts_kernel, dim3((B + 255) / 256), dim3(256), 0, (hipStream_t)stream, past, (const int4*)seqs, B, rows, longest);
  return check_launch(me);
}

static __global__ __launch_bounds__(256) void cache_advance_kernel(int* past, int B, int cap) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b >= B) return;
  const int p = past[b];
  if (p >= 0 && p < cap) past[b] = p + 1;
}

extern "C" int oat_window_cache_advance(int* past, int B, int cap, void* stream) {
  const char* me = "window_cache_advance";
  if (B < 0) return fail(me, "a negative number of sequences");
  if (B == 0) return 0;
  if (!past) return fail(me, "the counts are missing");
  OAT_LAUNCH(cache_advance_kernel, dim3((B + 255) / 256), dim3(256), 0, (hipStream_t)stream, past, B, cap < 0 ? 0x7fffffff : cap);
  return check_launch(me);
}

// ---- what a layer on packed q | k | v rows does, in one call each way (one crossing into the library instead of three).  The turned q and k
// are held in the rows' type: the matrix unit takes no more, and the cache keeps the keys as they are

// whether the gradient's way back through the rotary positions is taken where dq and dk are formed.  A pair's two values have to meet in one
// lane: those of a head's two halves do, in one register of two fragments, and this is the ladder that has the code.  (So would neighbours,
// and halves of fewer pairs that are a multiple of 8: such ladders take a pass of their own and round twice.)
static bool turns_in_halves(const OatRope* rope, int D) { return !rope->interleaved && 2 * rope->n_pairs == D; }
static int packed_wrong(const char* me, const OatRope* rope, const void* turned, int M, int Hq, int Hkv) {
  if (rope && !turned && M) return fail(me, "rotary positions need a buffer for the turned queries and keys");
  if (M < 0 || Hq < 1 || Hkv < 1) return fail(me, "no heads, or a negative number of rows");
  return 0;
}

static int layer_fwd(const void* qkv, long long ld, void* turned, float* table, const OatRope* rope, const int* pos, int period, void* out,
                                        float* lse, const int* seqs, int B, int longest, int M, int Hq, int Hkv, int D, int dtype, int left,
                                        int right, int sinks, float scale, void* kc, void* vc, const long long* strides, int cap, int clear, void* stream) {
  if (int rc = packed_wrong("window_attention_fwd", rope, turned, M, Hq, Hkv)) return rc;
  const long long n = (long long)(Hq + Hkv) * D, a = (long long)Hq * D;
  const char* q = (const char*)qkv;
  const char* v = M ? q + n * 2 : q;
  long long ldq = ld;
  if (rope) {
    if (int rc = rope_axes(qkv, ld, turned, n, dtype, pos, period, M, Hq + Hkv, D, rope, 0, (float2*)table, stream)) return rc;
    q = (const char*)turned;
    ldq = n;
  }
  const char* k = M ? q + a * 2 : q;
  if (int rc = attn_window_fwd(q, ldq, k, ldq, v, ld, out, a, lse, seqs, B, longest, longest, M, M, Hq, Hkv, D, dtype, left, right, sinks,
                               scale, clear, stream)) return rc;
  return kc ? cache_fill(k, ldq, v, ld, seqs, B, M, longest, M, longest, kc, vc, strides, cap, Hkv, D, sinks, stream) : 0;
}

static int layer_bwd(const void* qkv, long long ld, const void* turned, const float* table, const OatRope* rope, const int* pos, int period,
                                        const void* out, const float* lse, const void* dout, void* dqkv, const int* seqs, int B, int longest,
                                        int M, int Hq, int Hkv, int D, int dtype, int left, int right, int sinks, float scale, void* workspace,
                                        size_t workspace_bytes, int clear, void* stream) {
  if (int rc = packed_wrong("window_attention_bwd", rope, turned, M, Hq, Hkv)) return rc;
  if (M == 0) return 0;
  const long long n = (long long)(Hq + Hkv) * D, a = (long long)Hq * D, w = n + (long long)Hkv * D;
  const char* q = (const char*)(rope ? turned : qkv);
  const long long ldq = rope ? n : ld;
  char* g = (char*)dqkv;
  // turned back where they are formed, before their one rounding; a pass of its own rounds twice.  (A training pass of 32 captions
  // 134 -> 127 us, of two 16-frame clips 446 -> 436, of six packed texts with heads of 128 287 -> 286)
  const float2* turns = rope && table && turns_in_halves(rope, D) ? (const float2*)table : nullptr;
  if (turns && (uintptr_t)table % 8) return fail("window_attention_bwd", "the table of the turns is not aligned to 8 bytes");
  if (int rc = attn_window_bwd(q, ldq, q + a * 2, ldq, (const char*)qkv + n * 2, ld, out, a, lse, dout, a, g, w, g + a * 2, w, g + n * 2, w,
                                   seqs, B, longest, longest, M, M, Hq, Hkv, D, dtype, left, right, sinks, scale, workspace, workspace_bytes,
                               turns, clear, stream)) return rc;
  return rope && !turns ? oat_rope_axes(g, w, g, w, dtype, pos, period, M, Hq + Hkv, D, rope, 1, stream) : 0;
}

extern "C" int oat_window_attention_fwd(const void* qkv, long long ld, void* turned, float* table, const OatRope* rope, const int* pos, int period, void* out,
                                        float* lse, const int* seqs, int B, int longest, int M, int Hq, int Hkv, int D, int dtype, int left,
                                        int right, int sinks, float scale, void* kc, void* vc, const long long* strides, int cap, void* stream) {
  return layer_fwd(qkv, ld, turned, table, rope, pos, period, out, lse, seqs, B, longest, M, Hq, Hkv, D, dtype, left, right, sinks, scale, kc, vc, strides,
                   cap, 0, stream);
}
extern "C" int oat_window_attention_packed_fwd(const void* qkv, long long ld, void* turned, float* table, const OatRope* rope, const int* pos, int period, void* out,
                                        float* lse, const int* seqs, int B, int longest, int M, int Hq, int Hkv, int D, int dtype, int left,
                                        int right, int sinks, float scale, void* kc, void* vc, const long long* strides, int cap, void* stream) {
  return layer_fwd(qkv, ld, turned, table, rope, pos, period, out, lse, seqs, B, longest, M, Hq, Hkv, D, dtype, left, right, sinks, scale, kc, vc, strides,
                   cap, 1, stream);
}
extern "C" int oat_window_attention_bwd(const void* qkv, long long ld, const void* turned, const float* table, const OatRope* rope, const int* pos, int period,
                                        const void* out, const float* lse, const void* dout, void* dqkv, const int* seqs, int B, int longest,
                                        int M, int Hq, int Hkv, int D, int dtype, int left, int right, int sinks, float scale, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  return layer_bwd(qkv, ld, turned, table, rope, pos, period, out, lse, dout, dqkv, seqs, B, longest, M, Hq, Hkv, D, dtype, left, right, sinks, scale,
                   workspace, workspace_bytes, 0, stream);
}
extern "C" int oat_window_attention_packed_bwd(const void* qkv, long long ld, const void* turned, const float* table, const OatRope* rope, const int* pos, int period,
                                        const void* out, const float* lse, const void* dout, void* dqkv, const int* seqs, int B, int longest,
                                        int M, int Hq, int Hkv, int D, int dtype, int left, int right, int sinks, float scale, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  return layer_bwd(qkv, ld, turned, table, rope, pos, period, out, lse, dout, dqkv, seqs, B, longest, M, Hq, Hkv, D, dtype, left, right, sinks, scale,
                   workspace, workspace_bytes, 1, stream);
}
