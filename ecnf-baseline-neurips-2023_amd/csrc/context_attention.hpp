// context_attention.hpp — cross attention of a molecule's atoms to context states of another length (gfx950), forward
// and backward.
//
//   S = scale q k^T over the keys a row may read,  P = softmax(S),  O = P V,  lse = log sum exp S
//   delta = sum_d dO O,  dV = P^T dO,  dS = P (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q
//
// Rows.  The query heads that share one key head, and (where the whole batch reads one context) all molecules of the
// batch, are rows of the same product: row r of (context, key head) is query token t = r / G, head g = r % G, and
// t = molecule * n_queries + token.  So shared heads and a shared context cost no second read of K and V, a single token
// fills G rows of a tile, and the sums of dK and dV over a group's heads and over the batch happen in the accumulators.
//
// Products run on the 32x32 matrix instructions with the scores TRANSPOSED (keys down, rows across): in the
// accumulator layout lane l holds column l % 32 and the 16 rows (i & 3) + 8 (i >> 2) + 4 (l / 32), so one lane holds
// scores of one query row only.  Row maxima and sums are then in-lane (plus one exchange of the wave's halves), the
// running rescale is one scalar a lane, and the accumulator registers 8 s .. 8 s + 7 ARE the B operand of the next
// product's 16-key step if its A operand lists the keys in the same order ({4h .. 4h+3, 8+4h .. 8+4h+3}, h = l / 32):
// P never passes through LDS.  That A operand (V^T, or K^T / Q^T / dO^T in the backward pass) is read from the
// row-major LDS tile by the transposing LDS read (16-bit types) or column-wise (fp32).
//
// Types: bf16, fp16 (one 32x32x16 instruction a step) and fp32 (eight 32x32x2 instructions on the same fragments: the
// k order inside a step is free as long as A and B agree).  Scores, softmax statistics and all accumulators are fp32;
// P and dS are rounded to the operand type for the second products (half a step of the type, 2^-9 / 2^-12 relative,
// independent from key to key, so it averages in the sums).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace ecnf_ctx {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

#define ECNF_LDS(T) __attribute__((address_space(3))) T

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// n / d for n < 2^31 by one multiplication (d fixed for the launch)
struct FastDiv {
  uint32_t m, s, d;
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

// One launch's problem; strides in elements, last dimension contiguous, every row start 16-byte aligned.
struct Att {
  const char *q, *k, *v, *dout;
  char *out, *dq, *dk, *dv;
  float *lse;                      // [batch, heads, n_queries], natural log; NULL in the forward pass: not wanted
  float *part, *part_lse;          // split partials: [split][rows or keys, ...] (fp32)
  float *row_lse, *row_delta;      // backward: [context][key head][row], log2 units
  const int32_t *qlen, *klen;
  const uint8_t* mask;             // [contexts, keys], 0: masked
  int64_t qs[3], ks[3], vs[3], ds[3];
  FastDiv dG, dL;                  // rows -> token, token -> molecule
  int32_t B, C, Lq, Lk, Hq, Hk, D, G;
  int32_t per;                     // molecules of a context (B / C)
  int32_t R;                       // rows of a (context, key head): per * Lq * G
  int32_t tiles;                   // row or key tiles of a (context, key head)
  int32_t splits;
  float scale;
};

template <class T>
struct Ops;
template <>
struct Ops<__bf16> {
  typedef bf16x8 Frag;
  typedef bf16x4 Quad;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ Quad tr(ECNF_LDS(char) * p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((ECNF_LDS(bf16x4)*)p);
  }
};
template <>
struct Ops<_Float16> {
  typedef f16x8 Frag;
  typedef f16x4 Quad;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ Quad tr(ECNF_LDS(char) * p) {
    typedef __fp16 h4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((ECNF_LDS(h4)*)p));
  }
};
template <>
struct Ops<float> {
  typedef f32x8 Frag;
  typedef f32x4 Quad;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

// registers 8 s .. 8 s + 7 of an accumulator as the B operand of a 16-row step, rounded to T
template <class T>
__device__ __forceinline__ typename Ops<T>::Frag to_frag(const f32x16& x, int s) {
  typename Ops<T>::Frag f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (T)x[8 * s + e];
  return f;
}

__device__ __forceinline__ float other_half(float x) {   // the value of lane ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A row-major tile in LDS, rows of DP elements, its 16-byte chunks swizzled inside a row: chunk c of row r sits at
// c ^ f(r).  f takes 16 rows to 16 different groups of 4 banks (64 banks: fragment reads, 16 lanes of 16 rows, meet no
// conflict) and 4 consecutive rows to 4 different groups of 16 banks (the transposing read: 4 rows x 64 bytes).
template <class T, int DP>
struct Tile {
  static constexpr int kRow = DP * (int)sizeof(T);   // bytes
  static constexpr int kChunks = kRow / 16;
  static constexpr int kPer = 16 / (int)sizeof(T);   // elements of a chunk
  static __device__ __forceinline__ int f(int r) {
    if constexpr (kChunks >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (kChunks == 8) return ((r & 2) << 1) | ((r >> 2) & 3);
    else return (r >> 2) & 3;
  }
  static __device__ __forceinline__ int at(int r, int c) { return r * kRow + ((c ^ f(r)) << 4); }

  // operand of a 16-deep step s: 8 elements 16 s + 8 h .. of row r
  static __device__ __forceinline__ typename Ops<T>::Frag frag(const char* t, int r, int s, int h) {
    typedef typename Ops<T>::Frag Frag;
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const Frag*>(t + at(r, 2 * s + h));
    } else {
      const f32x4 a = *reinterpret_cast<const f32x4*>(t + at(r, 4 * s + 2 * h));
      const f32x4 b = *reinterpret_cast<const f32x4*>(t + at(r, 4 * s + 2 * h + 1));
      return Frag{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }
  // operand of the transposed product: column d0 + l % 32, rows r0 + {4h .. 4h+3, 8+4h .. 8+4h+3}
  static __device__ __forceinline__ typename Ops<T>::Frag frag_t(char* t, int r0, int d0, int l) {
    typename Ops<T>::Frag o;
    const int h = l >> 5;
    if constexpr (sizeof(T) == 2) {
      const int r = r0 + 4 * h + ((l & 15) >> 2), d = d0 + (l & 16) + 4 * (l & 3);
      const auto lo = Ops<T>::tr((ECNF_LDS(char)*)(t + at(r, d >> 3) + 2 * (d & 7)));
      const auto hi = Ops<T>::tr((ECNF_LDS(char)*)(t + at(r + 8, d >> 3) + 2 * (d & 7)));
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = lo[e], o[4 + e] = hi[e];
    } else {
      const int d = d0 + (l & 31);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int r = r0 + 4 * h + (e & 3) + 8 * (e >> 2);
        o[e] = *reinterpret_cast<const float*>(t + at(r, d >> 2) + 4 * (d & 3));
      }
    }
    return o;
  }
};

// block -> (tile, split, context and key head).  Consecutive blocks go to the 8 XCDs in turn; the blocks of one (context,
// key head) read the same K and V, so each XCD (with its own L2) takes a contiguous range of them.
__device__ __forceinline__ int xcd_order(int b, int n) {
  const int x = b & 7, i = b >> 3, q = n >> 3, rem = n & 7;
  return x * q + min(x, rem) + i;
}

__device__ __forceinline__ int key_count(const Att& a, int c) {
  return a.klen ? max(0, min(a.klen[c], a.Lk)) : a.Lk;
}

// row r of context c -> its molecule and token (r < R)
__device__ __forceinline__ void row_of(const Att& a, int c, int r, int& b, int& i, int& g) {
  const int t = (int)a.dG.div((uint32_t)r);
  g = r - t * a.G;
  const int m = a.per == 1 ? 0 : (int)a.dL.div((uint32_t)t);
  i = t - m * a.Lq;
  b = c * a.per + m;
}
__device__ __forceinline__ bool row_live(const Att& a, int b, int i) { return !a.qlen || i < a.qlen[b]; }

// The rows [r0, r0 + ROWS) of an operand as 16-byte chunks, NT threads: global -> registers -> LDS tile.  Rows outside
// their range (and masked keys) are zeros whatever memory holds there, so NaN or infinity behind a mask never enters a
// product; columns behind D (padding to the tile's DP) are zeros too.
template <class T, int DP, int ROWS, int NT>
struct Stage {
  static constexpr int kCh = Tile<T, DP>::kChunks;
  static constexpr int kN = (ROWS * kCh + NT - 1) / NT;
  u32x4 x[kN];
  template <class Addr>
  __device__ __forceinline__ void load(int tid, int D, Addr addr) {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int id = tid + n * NT, r = id / kCh, c = id % kCh;
      const char* p = (ROWS * kCh % NT == 0 || r < ROWS) && c * Tile<T, DP>::kPer < D ? addr(r) : nullptr;
      x[n] = u32x4{0, 0, 0, 0};
      if (p) x[n] = *reinterpret_cast<const u32x4*>(p + c * 16);
    }
  }
  __device__ __forceinline__ void store(char* t, int tid) const {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int id = tid + n * NT, r = id / kCh, c = id % kCh;
      if (ROWS * kCh % NT == 0 || r < ROWS) *reinterpret_cast<u32x4*>(t + Tile<T, DP>::at(r, c)) = x[n];
    }
  }
};

// 8-element fragments of row r's chunk straight from memory (the operands that stay in registers)
template <class T>
__device__ __forceinline__ typename Ops<T>::Frag frag_global(const char* row, int s, int h, int D) {
  typename Ops<T>::Frag f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (T)0.0f;
  const int d = 16 * s + 8 * h;
  if (row && d < D) {   // D % 8 == 0
    if constexpr (sizeof(T) == 2) {
      f = *reinterpret_cast<const typename Ops<T>::Frag*>(row + 2 * d);
    } else {
      const f32x4 a = *reinterpret_cast<const f32x4*>(row + 4 * d), b = *reinterpret_cast<const f32x4*>(row + 4 * d + 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = a[e], f[4 + e] = b[e];
    }
  }
  return f;
}

template <class T>
__device__ __forceinline__ void store4(char* p, f32x4 v) {
  typename Ops<T>::Quad o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = (T)v[e];
  *reinterpret_cast<typename Ops<T>::Quad*>(p) = o;
}

// ---------------------------------------------------------------------------------------------------------------
// forward.  A workgroup of 4 waves: WR of them split the rows (32 each), WK the keys of a tile (KT each); the waves of
// one row block join their statistics and outputs through LDS at the end.  grid = contexts * key heads * tiles * splits;
// with splits > 1 a workgroup takes its share of the key tiles and leaves a normalised fp32 partial and its lse.
// ---------------------------------------------------------------------------------------------------------------
template <class T, int DP, int WR, int WK, int KT>
struct FwdShape {
  static constexpr int kKeys = WK * KT;
  static constexpr int kTileBytes = kKeys * DP * (int)sizeof(T);
  static constexpr int kJoin = WK > 1 ? 4 * 32 * DP * 4 + 4 * 64 * 4 : 0;   // O of every wave, then m and l
  static constexpr int kLds = (2 * kTileBytes + kKeys * 4 > kJoin ? 2 * kTileBytes + kKeys * 4 : kJoin);
};

template <class T, int DP, int WR, int WK, int KT>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 1 : 2) void att_fwd(Att a) {
  typedef Tile<T, DP> TL;
  typedef FwdShape<T, DP, WR, WK, KT> Sh;
  constexpr int kKeys = Sh::kKeys, NS = DP / 16, ND = DP / 32, NB = KT / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char *kt = lds, *vt = lds + Sh::kTileBytes;
  float* bias = reinterpret_cast<float*>(lds + 2 * Sh::kTileBytes);
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6, h = l >> 5, wr = w % WR, wk = w / WR;
  int id = xcd_order(blockIdx.x, gridDim.x);
  const int tile = id % a.tiles;
  id /= a.tiles;
  const int split = id % a.splits;
  id /= a.splits;
  const int hk = id % a.Hk, c = id / a.Hk;

  const int r = tile * 32 * WR + wr * 32 + (l & 31);
  int b = 0, i = 0, g = 0;
  bool live = r < a.R;
  if (live) {
    row_of(a, c, r, b, i, g);
    live = row_live(a, b, i);
  }
  const char* qrow = live ? a.q + ((int64_t)b * a.qs[0] + (int64_t)i * a.qs[1] + (int64_t)(hk * a.G + g) * a.qs[2]) * (int64_t)sizeof(T)
                          : nullptr;
  typename Ops<T>::Frag qf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) qf[s] = frag_global<T>(qrow, s, h, a.D);

  const int n = key_count(a, c);
  const int nt = (n + kKeys - 1) / kKeys, share = (nt + a.splits - 1) / a.splits;
  const int t0 = min(split * share, nt), t1 = min(t0 + share, nt);
  const char* kb = a.k + ((int64_t)c * a.ks[0] + (int64_t)hk * a.ks[2]) * (int64_t)sizeof(T);
  const char* vb = a.v + ((int64_t)c * a.vs[0] + (int64_t)hk * a.vs[2]) * (int64_t)sizeof(T);
  const uint8_t* mask = a.mask ? a.mask + (int64_t)c * a.Lk : nullptr;
  auto allowed = [&](int key) { return key < n && (!mask || mask[key]); };

  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f32x16{};
  float m = -kInf, sum = 0.f;
  const float sc = a.scale * kLog2e;

  Stage<T, DP, kKeys, 256> sk, sv;
  auto fetch = [&](int t) {
    const int k0 = t * kKeys;
    sk.load(tid, a.D, [&](int x) { return allowed(k0 + x) ? kb + (int64_t)(k0 + x) * a.ks[1] * (int64_t)sizeof(T) : nullptr; });
    sv.load(tid, a.D, [&](int x) { return allowed(k0 + x) ? vb + (int64_t)(k0 + x) * a.vs[1] * (int64_t)sizeof(T) : nullptr; });
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    const bool whole = !mask && (t + 1) * kKeys <= n;
    __syncthreads();
    sk.store(kt, tid);
    sv.store(vt, tid);
    if (!whole && tid < kKeys) bias[tid] = allowed(t * kKeys + tid) ? 0.f : -kInf;
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);

    f32x16 sx[NB];
#pragma unroll
    for (int kb2 = 0; kb2 < NB; ++kb2) {
      sx[kb2] = f32x16{};
#pragma unroll
      for (int s = 0; s < NS; ++s)
        sx[kb2] = Ops<T>::mma(TL::frag(kt, wk * KT + kb2 * 32 + (l & 31), s, h), qf[s], sx[kb2]);
    }
    float mx = -kInf;
    if (!whole) {
#pragma unroll
      for (int kb2 = 0; kb2 < NB; ++kb2)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4 bs = *reinterpret_cast<const f32x4*>(bias + wk * KT + kb2 * 32 + 8 * j + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) sx[kb2][4 * j + e] = fmaf(sx[kb2][4 * j + e], sc, bs[e]);
        }
    } else {
#pragma unroll
      for (int kb2 = 0; kb2 < NB; ++kb2)
#pragma unroll
        for (int e = 0; e < 16; ++e) sx[kb2][e] *= sc;
    }
#pragma unroll
    for (int kb2 = 0; kb2 < NB; ++kb2)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sx[kb2][e]);
    mx = max_halves(mx);
    const float mn = fmaxf(m, mx);
    const float ref = mn == -kInf ? 0.f : mn;   // nothing allowed yet: exp2(-inf - 0) = 0
    if (__any(mn > m)) {
      const float al = __builtin_amdgcn_exp2f(m - ref);
      sum *= al;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= al;
      m = mn;
    }
#pragma unroll
    for (int kb2 = 0; kb2 < NB; ++kb2) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        sx[kb2][e] = __builtin_amdgcn_exp2f(sx[kb2][e] - ref);
        sum += sx[kb2][e];
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const auto p = to_frag<T>(sx[kb2], s);
#pragma unroll
        for (int d = 0; d < ND; ++d)
          o[d] = Ops<T>::mma(TL::frag_t(vt, wk * KT + kb2 * 32 + 16 * s, 32 * d, l), p, o[d]);
      }
    }
  }
  sum = sum_halves(sum);

  // ---- join the key waves, normalise, store.  lse in log2 units; an empty row has sum 0: output 0, lse -inf
  const int64_t grow = ((int64_t)c * a.Hk + hk) * a.R + r;
  auto put = [&](int rr, bool lv, int bb, int ii, int gg, int d, f32x4 v) {
    if (!lv) v = f32x4{0.f, 0.f, 0.f, 0.f};   // a row behind its molecule's length
    if (a.splits > 1) {
      if (rr < a.R)
        *reinterpret_cast<f32x4*>(a.part + (((int64_t)split * a.C * a.Hk + (int64_t)c * a.Hk + hk) * a.R + rr) * a.D + d) = v;
    } else if (rr < a.R) {
      store4<T>(a.out + ((((int64_t)bb * a.Lq + ii) * a.Hq + hk * a.G + gg) * a.D + d) * (int64_t)sizeof(T), v);
    }
  };
  if constexpr (WK == 1) {
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);   // NaN stays
    if (r < a.R) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int dd = 32 * d + 8 * j + 4 * h;
          if (dd < a.D)
            put(r, live, b, i, g, dd,
                f32x4{o[d][4 * j] * inv, o[d][4 * j + 1] * inv, o[d][4 * j + 2] * inv, o[d][4 * j + 3] * inv});
        }
      if (h == 0) {
        const float lse = sum == 0.f || !live ? -kInf : m + __builtin_amdgcn_logf(sum);
        if (a.splits > 1) a.part_lse[(int64_t)split * a.C * a.Hk * a.R + grow] = lse;
        else if (a.lse) a.lse[((int64_t)b * a.Hq + hk * a.G + g) * a.Lq + i] = lse * kLn2;
      }
    }
  } else {
    float* jo = reinterpret_cast<float*>(lds);                 // [wave][row][DP], 16-byte chunks swizzled by row
    float* jm = jo + 4 * 32 * DP;                              // [wave][row]
    float* jl = jm + 4 * 32;
    __syncthreads();
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(reinterpret_cast<char*>(jo + w * 32 * DP) + Tile<float, DP>::at(l & 31, 8 * d + 2 * j + h)) =
            f32x4{o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]};
    if (h == 0) jm[w * 32 + (l & 31)] = m, jl[w * 32 + (l & 31)] = sum;
    __syncthreads();
    for (int x = tid; x < WR * 32 * (DP / 4); x += 256) {
      const int ch = x % (DP / 4), row = x / (DP / 4), rw = row >> 5, rl = row & 31;
      const int rr = tile * 32 * WR + row;
      if (rr >= a.R || ch * 4 >= a.D) continue;
      float M = -kInf;
#pragma unroll
      for (int k = 0; k < WK; ++k) M = fmaxf(M, jm[(k * WR + rw) * 32 + rl]);
      const float ref = M == -kInf ? 0.f : M;
      float L = 0.f;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < WK; ++k) {
        const int ww = k * WR + rw;
        const float e = __builtin_amdgcn_exp2f(jm[ww * 32 + rl] - ref);
        L += e * jl[ww * 32 + rl];
        const f32x4 y = *reinterpret_cast<const f32x4*>(reinterpret_cast<const char*>(jo + ww * 32 * DP) + Tile<float, DP>::at(rl, ch));
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = fmaf(e, y[q], v[q]);
      }
      const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] *= inv;
      int bb, ii, gg;
      row_of(a, c, rr, bb, ii, gg);
      const bool lv = row_live(a, bb, ii);
      put(rr, lv, bb, ii, gg, ch * 4, v);
      if (ch == 0) {
        const float lse = L == 0.f || !lv ? -kInf : M + __builtin_amdgcn_logf(L);
        if (a.splits > 1) a.part_lse[((int64_t)split * a.C * a.Hk + (int64_t)c * a.Hk + hk) * a.R + rr] = lse;
        else if (a.lse) a.lse[((int64_t)bb * a.Hq + hk * a.G + gg) * a.Lq + ii] = lse * kLn2;
      }
    }
  }
}

// joins the splits of the forward pass: out = sum_s 2^(lse_s - M) part_s / sum_s 2^(lse_s - M); a thread has 4 columns
template <class T>
__global__ __launch_bounds__(256) void att_fwd_join(Att a) {
  const int64_t n = (int64_t)a.C * a.Hk * a.R;
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int D4 = a.D / 4;
  const int64_t row = x / D4;
  if (row >= n) return;
  const int ch = (int)(x - row * D4);
  float M = -kInf;
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.part_lse[s * n + row]);
  const float ref = M == -kInf ? 0.f : M;
  float L = 0.f;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    const float e = __builtin_amdgcn_exp2f(a.part_lse[s * n + row] - ref);
    L += e;
    const f32x4 y = *reinterpret_cast<const f32x4*>(a.part + (s * n + row) * a.D + 4 * ch);
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = fmaf(e, y[q], v[q]);
  }
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
#pragma unroll
  for (int q = 0; q < 4; ++q) v[q] *= inv;
  const int64_t ck = row / a.R;
  const int r = (int)(row - ck * a.R), hk = (int)(ck % a.Hk), c = (int)(ck / a.Hk);
  int b, i, g;
  row_of(a, c, r, b, i, g);
  store4<T>(a.out + ((((int64_t)b * a.Lq + i) * a.Hq + hk * a.G + g) * a.D + 4 * ch) * (int64_t)sizeof(T), v);
  if (ch == 0 && a.lse) a.lse[((int64_t)b * a.Hq + hk * a.G + g) * a.Lq + i] = (L == 0.f ? -kInf : M + __builtin_amdgcn_logf(L)) * kLn2;
}

// ---------------------------------------------------------------------------------------------------------------
// backward, dQ: the forward pass's shape (rows in registers, key tiles through LDS).  S^T and dP^T = V dO^T in the
// transposed layout, so P and dS need one lse and one delta a lane, and dQ^T += K^T dS^T takes dS from its accumulator
// registers.  Also writes every row's delta and lse (log2 units; +inf for a row without keys, whose P is then 0) for
// the kernel below.
// ---------------------------------------------------------------------------------------------------------------
template <class T, int DP, int WR, int WK, int KT>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 1 : 2) void att_dq(Att a) {
  typedef Tile<T, DP> TL;
  typedef FwdShape<T, DP, WR, WK, KT> Sh;
  constexpr int kKeys = Sh::kKeys, NS = DP / 16, ND = DP / 32, NB = KT / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char *kt = lds, *vt = lds + Sh::kTileBytes;
  float* bias = reinterpret_cast<float*>(lds + 2 * Sh::kTileBytes);
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6, h = l >> 5, wr = w % WR, wk = w / WR;
  int id = xcd_order(blockIdx.x, gridDim.x);
  const int tile = id % a.tiles;
  id /= a.tiles;
  const int split = id % a.splits;
  id /= a.splits;
  const int hk = id % a.Hk, c = id / a.Hk;

  const int r = tile * 32 * WR + wr * 32 + (l & 31);
  int b = 0, i = 0, g = 0;
  bool live = r < a.R;
  if (live) {
    row_of(a, c, r, b, i, g);
    live = row_live(a, b, i);
  }
  const int hq = hk * a.G + g;
  constexpr int64_t e = (int64_t)sizeof(T);
  const char* qrow = live ? a.q + ((int64_t)b * a.qs[0] + (int64_t)i * a.qs[1] + (int64_t)hq * a.qs[2]) * e : nullptr;
  const char* drow = live ? a.dout + ((int64_t)b * a.ds[0] + (int64_t)i * a.ds[1] + (int64_t)hq * a.ds[2]) * e : nullptr;
  const char* orow = live ? a.out + (((int64_t)b * a.Lq + i) * a.Hq + hq) * a.D * e : nullptr;
  typename Ops<T>::Frag qf[NS], df[NS];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    qf[s] = frag_global<T>(qrow, s, h, a.D);
    df[s] = frag_global<T>(drow, s, h, a.D);
    const auto of = frag_global<T>(orow, s, h, a.D);
#pragma unroll
    for (int x = 0; x < 8; ++x) delta = fmaf((float)df[s][x], (float)of[x], delta);
  }
  delta = sum_halves(delta);
  const float sc = a.scale * kLog2e;
  float lse = kInf;
  if (live) {
    lse = a.lse[((int64_t)b * a.Hq + hq) * a.Lq + i] * kLog2e;
    if (lse == -kInf) lse = kInf;
  }
  if (split == 0 && wk == 0 && h == 0 && r < a.R) {
    const int64_t row = ((int64_t)c * a.Hk + hk) * a.R + r;
    a.row_lse[row] = lse;
    a.row_delta[row] = delta;
  }

  const int n = key_count(a, c);
  const int nt = (n + kKeys - 1) / kKeys, share = (nt + a.splits - 1) / a.splits;
  const int t0 = min(split * share, nt), t1 = min(t0 + share, nt);
  const char* kb = a.k + ((int64_t)c * a.ks[0] + (int64_t)hk * a.ks[2]) * e;
  const char* vb = a.v + ((int64_t)c * a.vs[0] + (int64_t)hk * a.vs[2]) * e;
  const uint8_t* mask = a.mask ? a.mask + (int64_t)c * a.Lk : nullptr;
  auto allowed = [&](int key) { return key < n && (!mask || mask[key]); };

  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
  Stage<T, DP, kKeys, 256> sk, sv;
  auto fetch = [&](int t) {
    const int k0 = t * kKeys;
    sk.load(tid, a.D, [&](int x) { return allowed(k0 + x) ? kb + (int64_t)(k0 + x) * a.ks[1] * e : nullptr; });
    sv.load(tid, a.D, [&](int x) { return allowed(k0 + x) ? vb + (int64_t)(k0 + x) * a.vs[1] * e : nullptr; });
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    const bool whole = !mask && (t + 1) * kKeys <= n;
    __syncthreads();
    sk.store(kt, tid);
    sv.store(vt, tid);
    if (!whole && tid < kKeys) bias[tid] = allowed(t * kKeys + tid) ? 0.f : -kInf;
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
#pragma unroll
    for (int kb2 = 0; kb2 < NB; ++kb2) {
      const int k0 = wk * KT + kb2 * 32;
      f32x16 sx = f32x16{}, dp = f32x16{};
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        sx = Ops<T>::mma(TL::frag(kt, k0 + (l & 31), s, h), qf[s], sx);
        dp = Ops<T>::mma(TL::frag(vt, k0 + (l & 31), s, h), df[s], dp);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 bs = {0.f, 0.f, 0.f, 0.f};
        if (!whole) bs = *reinterpret_cast<const f32x4*>(bias + k0 + 8 * j + 4 * h);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float p = __builtin_amdgcn_exp2f(fmaf(sx[4 * j + x], sc, bs[x] - lse));
          sx[4 * j + x] = p * (dp[4 * j + x] - delta);
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const auto dsf = to_frag<T>(sx, s);
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] = Ops<T>::mma(TL::frag_t(kt, k0 + 16 * s, 32 * d, l), dsf, acc[d]);
      }
    }
  }

  const int64_t n_rows = (int64_t)a.C * a.Hk * a.R, row0 = ((int64_t)c * a.Hk + hk) * a.R;
  auto put = [&](int rr, bool lv, int bb, int ii, int gg, int d, f32x4 v) {
    if (rr >= a.R) return;
    if (!lv) v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] *= a.scale;
    if (a.splits > 1) *reinterpret_cast<f32x4*>(a.part + (split * n_rows + row0 + rr) * a.D + d) = v;
    else store4<T>(a.dq + ((((int64_t)bb * a.Lq + ii) * a.Hq + hk * a.G + gg) * a.D + d) * e, v);
  };
  if constexpr (WK == 1) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int dd = 32 * d + 8 * j + 4 * h;
        if (dd < a.D) put(r, live, b, i, g, dd, f32x4{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]});
      }
  } else {
    float* jo = reinterpret_cast<float*>(lds);
    __syncthreads();
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(reinterpret_cast<char*>(jo + w * 32 * DP) + Tile<float, DP>::at(l & 31, 8 * d + 2 * j + h)) =
            f32x4{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
    __syncthreads();
    for (int x = tid; x < WR * 32 * (DP / 4); x += 256) {
      const int ch = x % (DP / 4), row = x / (DP / 4), rw = row >> 5, rl = row & 31;
      const int rr = tile * 32 * WR + row;
      if (rr >= a.R || ch * 4 >= a.D) continue;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < WK; ++k)
        v += *reinterpret_cast<const f32x4*>(reinterpret_cast<const char*>(jo + (k * WR + rw) * 32 * DP) + Tile<float, DP>::at(rl, ch));
      int bb, ii, gg;
      row_of(a, c, rr, bb, ii, gg);
      put(rr, row_live(a, bb, ii), bb, ii, gg, ch * 4, v);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// backward, dK and dV: a wave keeps 32 keys (K and V as B operands, both gradients as accumulators) and the row tiles
// pass through LDS.  S and dP have keys across, so P and dS are the B operands of dV^T += dO^T P and dK^T += Q^T dS as
// they stand.  WY waves split the keys of a workgroup, WX its rows (joined through LDS); with splits > 1 a workgroup
// takes its share of the row tiles and leaves fp32 partials.  The order of every sum is fixed.
// ---------------------------------------------------------------------------------------------------------------
template <class T, int DP, int WY, int WX>
struct DkvShape {
  static constexpr int kRows = 32 * WX;
  static constexpr int kTileBytes = kRows * DP * (int)sizeof(T);
  static constexpr int kLoop = 2 * kTileBytes + 2 * kRows * 4;
  static constexpr int kJoin = WX > 1 ? 4 * 32 * DP * 4 : 0;
  static constexpr int kLds = kLoop > kJoin ? kLoop : kJoin;
};

template <class T, int DP, int WY, int WX>
__global__ __launch_bounds__(256, 1) void att_dkv(Att a) {
  typedef Tile<T, DP> TL;
  typedef DkvShape<T, DP, WY, WX> Sh;
  constexpr int kRows = Sh::kRows, NS = DP / 16, ND = DP / 32;
  constexpr int64_t e = (int64_t)sizeof(T);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char *qt = lds, *dt = lds + Sh::kTileBytes;
  float* rl = reinterpret_cast<float*>(lds + 2 * Sh::kTileBytes);
  float* rd = rl + kRows;
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6, h = l >> 5, wy = w % WY, wx = w / WY;
  int id = xcd_order(blockIdx.x, gridDim.x);
  const int tile = id % a.tiles;
  id /= a.tiles;
  const int split = id % a.splits;
  id /= a.splits;
  const int hk = id % a.Hk, c = id / a.Hk;

  const int n = key_count(a, c);
  const int key = (tile * WY + wy) * 32 + (l & 31);
  const uint8_t* mask = a.mask ? a.mask + (int64_t)c * a.Lk : nullptr;
  const bool ok = key < n && (!mask || mask[key]);
  const char* krow = ok ? a.k + ((int64_t)c * a.ks[0] + (int64_t)key * a.ks[1] + (int64_t)hk * a.ks[2]) * e : nullptr;
  const char* vrow = ok ? a.v + ((int64_t)c * a.vs[0] + (int64_t)key * a.vs[1] + (int64_t)hk * a.vs[2]) * e : nullptr;
  typename Ops<T>::Frag kf[NS], vf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) kf[s] = frag_global<T>(krow, s, h, a.D), vf[s] = frag_global<T>(vrow, s, h, a.D);
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dk[d] = f32x16{}, dv[d] = f32x16{};

  // no key of the workgroup is inside its context: nothing to sum (the rows loop is uniform over the workgroup)
  const int nt = tile * WY * 32 < n ? (a.R + kRows - 1) / kRows : 0, share = (nt + a.splits - 1) / a.splits;
  const int t0 = min(split * share, nt), t1 = min(t0 + share, nt);
  const int64_t row0 = ((int64_t)c * a.Hk + hk) * a.R;
  const float sc = a.scale * kLog2e;

  Stage<T, DP, kRows, 256> sq, sd;
  float nl = kInf, nd = 0.f;
  auto fetch = [&](int t) {
    const int r0 = t * kRows;
    sq.load(tid, a.D, [&](int x) -> const char* {
      if (r0 + x >= a.R) return nullptr;
      int b, i, g;
      row_of(a, c, r0 + x, b, i, g);
      if (!row_live(a, b, i)) return nullptr;
      return a.q + ((int64_t)b * a.qs[0] + (int64_t)i * a.qs[1] + (int64_t)(hk * a.G + g) * a.qs[2]) * e;
    });
    sd.load(tid, a.D, [&](int x) -> const char* {
      if (r0 + x >= a.R) return nullptr;
      int b, i, g;
      row_of(a, c, r0 + x, b, i, g);
      if (!row_live(a, b, i)) return nullptr;
      return a.dout + ((int64_t)b * a.ds[0] + (int64_t)i * a.ds[1] + (int64_t)(hk * a.G + g) * a.ds[2]) * e;
    });
    if (tid < kRows) {
      const bool in = r0 + tid < a.R;
      nl = in ? a.row_lse[row0 + r0 + tid] : kInf;
      nd = in ? a.row_delta[row0 + r0 + tid] : 0.f;
    }
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    __syncthreads();
    sq.store(qt, tid);
    sd.store(dt, tid);
    if (tid < kRows) rl[tid] = nl, rd[tid] = nd;
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
    const int x0 = wx * 32;
    f32x16 sx = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      sx = Ops<T>::mma(TL::frag(qt, x0 + (l & 31), s, h), kf[s], sx);
      dp = Ops<T>::mma(TL::frag(dt, x0 + (l & 31), s, h), vf[s], dp);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4 ls = *reinterpret_cast<const f32x4*>(rl + x0 + 8 * j + 4 * h);
      const f32x4 de = *reinterpret_cast<const f32x4*>(rd + x0 + 8 * j + 4 * h);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float p = __builtin_amdgcn_exp2f(fmaf(sx[4 * j + x], sc, -ls[x]));
        p = ok ? p : 0.f;
        sx[4 * j + x] = p;
        dp[4 * j + x] = p * (dp[4 * j + x] - de[x]);
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const auto pf = to_frag<T>(sx, s), sf = to_frag<T>(dp, s);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        dv[d] = Ops<T>::mma(TL::frag_t(dt, x0 + 16 * s, 32 * d, l), pf, dv[d]);
        dk[d] = Ops<T>::mma(TL::frag_t(qt, x0 + 16 * s, 32 * d, l), sf, dk[d]);
      }
    }
  }

  const int64_t n_keys = (int64_t)a.C * a.Hk * a.Lk;
  auto put = [&](int which, int kk, int d, f32x4 v) {
    if (kk >= a.Lk || d >= a.D) return;
    if (which == 0)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] *= a.scale;
    if (a.splits > 1) {
      *reinterpret_cast<f32x4*>(a.part + (((int64_t)split * 2 + which) * n_keys + ((int64_t)c * a.Hk + hk) * a.Lk + kk) * a.D + d) = v;
    } else {
      store4<T>((which ? a.dv : a.dk) + ((((int64_t)c * a.Lk + kk) * a.Hk + hk) * a.D + d) * e, v);
    }
  };
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const f32x16* acc = which ? dv : dk;
    if constexpr (WX == 1) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          put(which, key, 32 * d + 8 * j + 4 * h, f32x4{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]});
    } else {
      float* jo = reinterpret_cast<float*>(lds);
      __syncthreads();
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<f32x4*>(reinterpret_cast<char*>(jo + w * 32 * DP) + Tile<float, DP>::at(l & 31, 8 * d + 2 * j + h)) =
              f32x4{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
      __syncthreads();
      for (int x = tid; x < WY * 32 * (DP / 4); x += 256) {
        const int ch = x % (DP / 4), kr = x / (DP / 4), ky = kr >> 5, kl = kr & 31;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < WX; ++q)
          v += *reinterpret_cast<const f32x4*>(reinterpret_cast<const char*>(jo + (q * WY + ky) * 32 * DP) + Tile<float, DP>::at(kl, ch));
        put(which, (tile * WY + ky) * 32 + kl, ch * 4, v);
      }
    }
  }
}

// sums the splits' partials (in order): which = 0 dQ rows, 1 dK and dV keys (blockIdx.y: 0 dK, 1 dV); 4 columns a thread
template <class T>
__global__ __launch_bounds__(256) void att_grad_join(Att a, int which) {
  const int D4 = a.D / 4;
  const int64_t n = (int64_t)a.C * a.Hk * (which ? a.Lk : a.R);
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = x / D4;
  if (row >= n) return;
  const int d = 4 * (int)(x - row * D4);
  const int kinds = which ? 2 : 1, y = which ? (int)blockIdx.y : 0;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s)
    v += *reinterpret_cast<const f32x4*>(a.part + (((int64_t)s * kinds + y) * n + row) * a.D + d);
  const int len = which ? a.Lk : a.R;
  const int64_t ck = row / len;
  const int r = (int)(row - ck * len), hk = (int)(ck % a.Hk), c = (int)(ck / a.Hk);
  char* p;
  if (which) {
    p = (y ? a.dv : a.dk) + ((((int64_t)c * a.Lk + r) * a.Hk + hk) * a.D + d) * (int64_t)sizeof(T);
  } else {
    int b, i, g;
    row_of(a, c, r, b, i, g);
    p = a.dq + ((((int64_t)b * a.Lq + i) * a.Hq + hk * a.G + g) * a.D + d) * (int64_t)sizeof(T);
  }
  store4<T>(p, v);
}

// ---------------------------------------------------------------------------------------------------------------
// launch plans (the same on the sizing and the launching side)
// ---------------------------------------------------------------------------------------------------------------
// the split partials of one kernel are at most this many floats (256 MiB)
constexpr int64_t kPartMax = 64ll << 20;

struct Plan {
  int narrow;    // 1: the waves split the inner dimension (few rows / few keys), 0: the outer one
  int tiles, splits;
  int64_t grid, part, part_lse;   // workgroups; workspace floats
};

inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// outer: rows (forward, dQ) or keys (dK dV) of a (context, key head), `inner` the loop's length in elements of
// `step(narrow)`; per_row: partial floats of one outer element and split.
inline Plan make_plan(int64_t pairs, int outer, int inner, int narrow_step, int wide_step, int64_t per_row, bool lse) {
  Plan p;
  p.narrow = outer <= 32;
  p.tiles = ceil_div(outer, p.narrow ? 32 : 128);
  const int64_t base = pairs * p.tiles;
  const int inner_tiles = ceil_div(inner, p.narrow ? narrow_step : wide_step);
  int64_t s = 1;
  if (base > 0 && base < 512) s = (512 + base - 1) / base;
  if (s > inner_tiles / 4) s = inner_tiles / 4;
  const int64_t one = pairs * outer * per_row;
  if (one > 0 && s * one > kPartMax) s = kPartMax / one;
  p.splits = (int)(s < 1 ? 1 : s);
  p.grid = base * p.splits;
  p.part = p.splits > 1 ? (int64_t)p.splits * one : 0;
  p.part_lse = p.splits > 1 && lse ? (int64_t)p.splits * pairs * outer : 0;
  return p;
}
inline Plan plan_fwd(const Att& a) { return make_plan((int64_t)a.C * a.Hk, a.R, a.Lk, 128, 64, a.D, true); }
inline Plan plan_dq(const Att& a) { return make_plan((int64_t)a.C * a.Hk, a.R, a.Lk, 128, 64, a.D, false); }
inline Plan plan_dkv(const Att& a) { return make_plan((int64_t)a.C * a.Hk, a.Lk, a.R, 128, 32, 2 * a.D, false); }

// one per element type (ecnf_attention.hip)
hipError_t launch_fwd_bf16(const Att&, hipStream_t);
hipError_t launch_fwd_f16(const Att&, hipStream_t);
hipError_t launch_fwd_f32(const Att&, hipStream_t);
hipError_t launch_grad_bf16(const Att&, hipStream_t);
hipError_t launch_grad_f16(const Att&, hipStream_t);
hipError_t launch_grad_f32(const Att&, hipStream_t);

}  // namespace ecnf_ctx
