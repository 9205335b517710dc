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
// P and dS are rounded to the operand type for the second products (at most half a step, 2^-8 / 2^-11 relative, independent
// from key to key: with the outputs' own rounding 0.6 half steps in norm, where one rounding is 0.43).
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

// waves a SIMD: at least LOW (what the kernel's registers allow without spills); at head_dim 128 exactly that many, so
// that the scheduler spends the registers on reads ahead (long bf16 forward 1078 us, with as many as fit 1085), and
// elsewhere as many as fit (training pass of 22 x 129 at head_dim 16, exactly LOW: fp32 82 us for 74, bf16 46 for 43)
#define ECNF_WAVES(LOW) __attribute__((amdgpu_waves_per_eu((LOW), HD <= 64 ? 8 : (LOW))))
constexpr int waves(int hd, int bytes, int at32, int at64) {
  return bytes == 4 ? (hd <= 32 ? 3 : hd <= 64 ? 2 : 1) : hd <= 32 ? at32 : hd <= 64 ? at64 : 2;
}
// The kernels are compiled for head_dim up to HD = 16, 32, 64, 96 and 128 (steps of 16 in the scores, blocks of 32 in
// the outputs); LDS rows are the next power of two.
constexpr int tile_width(int hd) { return hd <= 32 ? 32 : hd <= 64 ? 64 : 128; }
#define ECNF_LDS(T) __attribute__((address_space(3))) T

template <int V>
struct Const {
  static constexpr int value = V;
};

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
  int32_t elem;                    // bytes of an element
  int32_t flat;                    // tokens of a context are one sequence in q and dout (see RowTile)
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
  static __device__ __forceinline__ Quad tr(uint32_t p) {
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
  static __device__ __forceinline__ Quad tr(uint32_t p) {
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

__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The backward pass in fp16.  P is about 1 / keys and dS smaller still, at or below fp16's subnormals in long contexts
// (1 / 16384 = 2^-14).  So P is made as 2^14 P (at most 2^14: a shift of the exponent's argument, for nothing), dS with
// it, and where the largest 2^14 |dS| of a column (row of dQ, key of dK) so far is not in [1, 2^15] the column is scaled
// by a power of two besides, which its accumulators carry.  What is rounded away is then 2^-11 of the value, or 2^-25 of
// the column's largest.  Other types have fp32's exponents and need nothing.
template <class T>
struct Range {
  static constexpr float kShift = 0.f, kBack = 1.f;
  __device__ __forceinline__ void fit(f32x16&, f32x16*, int) {}
  __device__ __forceinline__ float back() const { return 1.f; }
};
template <>
struct Range<_Float16> {
  static constexpr float kShift = 14.f, kBack = 0x1p-14f;
  float scale = 1.f, top = 0.f;
  // scales x (one column a lane, its other rows in the other half), and the accumulators where the scale moves
  __device__ __forceinline__ void fit(f32x16& x, f32x16* acc, int n) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(x[i]));
    top = fmaxf(top, max_halves(m));
    const float at = top * scale;
    const bool out = at > 32768.f || (at < 1.f && at > 0.f);
    if (__any(out)) {
      // the largest lands in [2^14, 2^15); an infinity or NaN stays one
      const uint32_t e = (uint32_t)min(max(268 - (int)(__float_as_uint(top) >> 23), 1), 254);
      const float next = out ? __uint_as_float(e << 23) : scale, move = next / scale;
      scale = next;
#pragma unroll
      for (int d = 0; d < n; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] *= move;
    }
    if (__any(scale != 1.f))
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] *= scale;
  }
  __device__ __forceinline__ float back() const { return kBack / scale; }
};

// A row-major tile in LDS, rows of DP elements, its 16-byte chunks swizzled inside a row: chunk c of row r sits at
// c ^ f(r).  f takes 16 rows to 16 different groups of 4 banks (64 banks: fragment reads, 16 lanes of 16 rows, meet no
// conflict) and 4 consecutive rows to 4 different groups of 16 banks (the transposing read: 4 rows x 64 bytes).
template <class T, int DP>
struct Tile {
  static constexpr int kRow = DP * (int)sizeof(T);   // bytes
  static constexpr int kChunks = kRow / 16;
  static constexpr int kPer = 16 / (int)sizeof(T);   // elements of a chunk
  static constexpr __host__ __device__ __forceinline__ int f(int r) {
    if constexpr (kChunks >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (kChunks == 8) return ((r & 2) << 1) | ((r >> 2) & 3);
    else return (r >> 2) & 3;
  }
  static __device__ __forceinline__ int at(int r, int c) { return r * kRow + ((c ^ f(r)) << 4); }
};

// A lane's reads of tiles.  f only permutes bits, so every address is the lane's base with constant bits turned
// (one instruction) plus a constant offset: nothing but two bases stays in registers.
template <class T, int DP>
struct Reader {
  typedef Tile<T, DP> TL;
  typedef typename Ops<T>::Frag Frag;
  uint32_t fb, tb;
  // l: lane; base: LDS address of the first tile (a multiple of 512, like every tile's)
  __device__ __forceinline__ void init(uint32_t base, int l) {
    const int h = l >> 5;
    if constexpr (sizeof(T) == 2) {
      fb = base + TL::at(l & 31, h);
      tb = base + TL::at(4 * h + ((l & 15) >> 2), ((l & 16) >> 3) | ((l & 3) >> 1)) + 8 * (l & 1);
    } else {
      fb = base + TL::at(l & 31, 2 * h);
      tb = base + TL::at(4 * h, (l & 31) >> 2) + 4 * (l & 3);
    }
  }
  // operand of a 16-deep step s: elements 16 s + 8 h .. + 7 of row r0 + l % 32 (r0 a multiple of 32) of the tile at `at`
  __device__ __forceinline__ Frag frag(uint32_t at, int r0, int s) const {
    if constexpr (sizeof(T) == 2) {
      return *(ECNF_LDS(const Frag)*)(((fb + at) ^ (uint32_t)(s << 5)) + r0 * TL::kRow);
    } else {
      const uint32_t p = ((fb + at) ^ (uint32_t)(s << 6)) + r0 * TL::kRow, q = ((fb + at) ^ (uint32_t)(s << 6 | 16)) + r0 * TL::kRow;
      const f32x4 x = *(ECNF_LDS(const f32x4)*)p, y = *(ECNF_LDS(const f32x4)*)q;
      return Frag{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    }
  }
  // operand of the transposed product: column 32 d + l % 32 of the rows r0 + {4h .. 4h+3, 8+4h .. 8+4h+3} (r0 % 16 = 0)
  __device__ __forceinline__ Frag frag_t(uint32_t at, int r0, int d) const {
    Frag o;
    if constexpr (sizeof(T) == 2) {
      const auto lo = Ops<T>::tr(((tb + at) ^ (uint32_t)(d << 6)) + r0 * TL::kRow);
      const auto hi = Ops<T>::tr(((tb + at) ^ (uint32_t)(d << 6 ^ TL::f(8) << 4)) + (r0 + 8) * TL::kRow);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = lo[e], o[4 + e] = hi[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int r = (e & 3) + 8 * (e >> 2);
        o[e] = *(ECNF_LDS(const float)*)(((tb + at) ^ (uint32_t)(d << 7 ^ TL::f(r) << 4)) + (r0 + r) * TL::kRow);
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
  return a.klen ? __builtin_amdgcn_readfirstlane(max(0, min(a.klen[c], a.Lk))) : a.Lk;
}

// Whether the first n keys of a context leave a row exactly one: then P is 1 whatever q and k are, and dS is 0.  By length,
// or by the mask (0: masked), where `some` is a ballot of keys that the wave knows to be allowed: two of them and the answer
// is there.  Else every wave counts for itself, 1024 keys at a time, until the second key.
__device__ __forceinline__ bool one_key(const uint8_t* mask, int n, int lane, uint64_t some) {
  if (!mask || n <= 1) return n == 1;
  if (__popcll(some) > 1) return false;
  int count = 0;
  for (int k0 = 0; k0 < n && count < 2; k0 += 1024) {
    uint8_t m[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int key = k0 + 64 * j + lane;
      m[j] = key < n ? mask[key] : (uint8_t)0;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) count += __popcll(__ballot(m[j] != 0));
  }
  return count == 1;
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

// Tiles go from memory to LDS without passing registers (16-byte LDS loads): a wave's 64 chunks land consecutively, so
// the lane that fills slot c' of row r asks for chunk c' ^ f(r).  Issued through asm (the compiler would otherwise make
// every later LDS read wait for them); dma_wait before the barrier that publishes them.
__device__ __forceinline__ u32x4 uniform(u32x4 x) {   // the same in every lane, so that it can sit in scalar registers
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_readfirstlane(x[i]);
  return x;
}
__device__ __forceinline__ void dma_buffer(uint32_t lds, u32x4 rsrc, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(rsrc)
               : "memory", "m0");
}
__device__ __forceinline__ void dma_global(uint32_t lds, const char* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(p) : "memory", "m0");
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(ECNF_LDS(const void)*)p; }
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// A tile of ROWS keys: constant stride, so one buffer descriptor a tile (its range ends behind the last valid row) and
// lane offsets that stay the same from tile to tile.  What lies behind the range reads as zero, and a masked key's lanes
// ask behind the range: NaN or infinity behind a length or mask never enters a product.  Columns behind D are zero too.
constexpr uint32_t kBehind = 0x80000000u;
template <class T, int DP, int ROWS>
struct KeyTile {
  static constexpr int kCh = Tile<T, DP>::kChunks;
  static constexpr int kN = ROWS * kCh / 256;       // chunks a thread
  static constexpr int kStep = 256 / kCh;           // rows from one to the next
  static constexpr int kAlt = kCh == 32 ? 2 : 1;    // f repeats every 16 rows
  static_assert(kN >= 1 && ROWS * kCh % 256 == 0 && kStep * kAlt % 16 == 0, "whole chunks of a workgroup");
  const char* base;
  uint32_t stride, off[kAlt];
  int row, end;   // end: bytes of a row
  __device__ __forceinline__ void init(const char* b, int64_t row_stride, int D, int tid) {
    base = b;
    stride = (uint32_t)row_stride;
    end = D * (int)sizeof(T);
    row = tid / kCh;
#pragma unroll
    for (int x = 0; x < kAlt; ++x) {
      const int c = ((tid % kCh) ^ Tile<T, DP>::f(row + x * kStep)) * 16;
      off[x] = c < end ? (row + x * kStep) * stride + c : kBehind;
    }
  }
  template <class Allowed>
  __device__ __forceinline__ void load(uint32_t lds, int k0, int valid, bool masked, Allowed allowed) const {
    const uint64_t p = (uint64_t)(base + (int64_t)k0 * stride);
    const int rows = min(valid, ROWS);
    const u32x4 rsrc = uniform(u32x4{(uint32_t)p, (uint32_t)(p >> 32) & 0xffffu, (uint32_t)(rows - 1) * stride + (uint32_t)end, 0x00020000u});
    const uint32_t at = lds + wave_id() * 1024;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      uint32_t o = off[n % kAlt] + (uint32_t)(n / kAlt * kAlt * kStep) * stride;
      if (masked) o = allowed(row + n * kStep) ? o : kBehind;
      dma_buffer(at + n * 4096, rsrc, o);
    }
  }
};

static __device__ const u32x4 kZeroRow[32] = {};   // 512 bytes: the longest row

// A tile of ROWS query rows.  Fast form: a tile is whole tokens (G divides ROWS), the tokens of a context are evenly
// spaced (a.flat) and none is behind a length, so like a key tile it is a descriptor that moves from tile to tile and
// fixed lane offsets; only rows behind the last one turn to zero.  General form: an address a row, zeros from kZeroRow.
template <class T, int DP, int ROWS>
struct RowTile {
  typedef Tile<T, DP> TL;
  static constexpr int kCh = TL::kChunks;
  static constexpr int kN = (ROWS * kCh + 255) / 256;
  static_assert(ROWS * kCh % 64 == 0, "whole chunks of a wave");
  const char* base;
  int64_t s0, s1, s2;   // bytes
  uint32_t off[kN];
  __device__ __forceinline__ static int row(int n, int tid) { return (tid + n * 256) / kCh; }
  __device__ __forceinline__ static bool mine(int n) { return ROWS * kCh % 256 == 0 || n * 256 + wave_id() * 64 < ROWS * kCh; }
  __device__ __forceinline__ void init(const Att& a, const char* p, const int64_t* st, int c, int hk, int tid, bool fast) {
    constexpr int64_t e = (int64_t)sizeof(T);
    s0 = st[0] * e, s1 = st[1] * e, s2 = st[2] * e;
    base = p + (int64_t)hk * a.G * s2 + (int64_t)c * a.per * s0;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int r = row(n, tid), ch = ((tid + n * 256) % kCh) ^ TL::f(r);
      const int t = (int)a.dG.div((uint32_t)r), g = r - t * a.G;
      const uint32_t o = (fast ? (uint32_t)t * (uint32_t)s1 + (uint32_t)g * (uint32_t)s2 : 0u) + ch * 16;
      off[n] = ch * TL::kPer < a.D ? o : kBehind;
    }
  }
  // rows r0 .. of context c into the tile at `lds`
  __device__ __forceinline__ void load(const Att& a, uint32_t lds, int c, int r0, int tid, bool fast) const {
    const uint32_t at = lds + wave_id() * 1024;
    if (fast) {
      const uint64_t p = (uint64_t)(base + (int64_t)a.dG.div((uint32_t)r0) * s1);
      const u32x4 rsrc = uniform(u32x4{(uint32_t)p, (uint32_t)(p >> 32) & 0xffffu, 0x7ffffff0u, 0x00020000u});
      const bool tail = r0 + ROWS > a.R;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        if (!mine(n)) break;
        uint32_t o = off[n];
        if (tail) o = r0 + row(n, tid) < a.R ? o : kBehind;
        dma_buffer(at + n * 4096, rsrc, o);
      }
    } else {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        if (!mine(n)) break;
        const int r = min(r0 + row(n, tid), a.R - 1);
        int b, i, g;
        row_of(a, 0, r, b, i, g);
        const bool ok = off[n] != kBehind && r0 + row(n, tid) < a.R && row_live(a, c * a.per + b, i);
        const char* x = base + (int64_t)b * s0 + (int64_t)i * s1 + (int64_t)g * s2 + off[n];
        dma_global(at + n * 4096, ok ? x : reinterpret_cast<const char*>(kZeroRow));
      }
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

// |scale| in log2 units.  0 becomes the smallest number, under which any finite score is at most 5e-7 (a factor of 0 would
// make NaN of a masked key's -inf)
__device__ __forceinline__ float log2_scale(float scale) { return fmaxf(fabsf(scale) * kLog2e, 0x1p-149f); }

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
//
// Long contexts are bound by the matrix units and the exponentials beside them (MFMA busy 0.51, vector 0.46 of a clock
// that falls to 1.83 GHz; no LDS bank conflict): 2 x 4096 queries of 32 heads on 8192 keys of 8, 128 wide, bf16, 1037 us,
// 1060 TFLOP/s (a library product of 8192^3: 1163).  So 32 rows a wave, tiles of 64 keys in two buffers with one barrier
// each; 64 rows a wave spill (1341 us), tiles of 32 pay the barrier twice (1106).  Single tokens are bound by reading
// K and V: 64 x 8192 keys of 8 x 128 in 376 us, 5.7 TB/s.  Small contexts by latency: 512 x 22 rows x 333 masked keys of
// 4 x 64, bf16, 30 us, 3.6 TB/s.
// ---------------------------------------------------------------------------------------------------------------
template <class T, int DP, int WR, int WK, int KT, int BUFS>
struct FwdShape {
  static constexpr int kKeys = WK * KT;
  static constexpr int kTileBytes = kKeys * DP * (int)sizeof(T);
  // two buffers of K, V and the keys' bias; where the waves split the keys, the join reuses them: O of every wave, m, l
  static constexpr int kBuf = 2 * kTileBytes;
  static constexpr int kBufs = BUFS * kBuf + 3 * kKeys * 4 <= 160 * 1024 ? BUFS : 1;
  static constexpr int kBias = kBufs * kBuf;   // the biases lie behind the tiles (which start on multiples of 512 bytes)
  static constexpr int kDelta = kBias + 3 * kKeys * 4;   // dQ: a sum a row and wave
  static constexpr int kLoop = kDelta + 4 * 32 * 4;
  static constexpr int kJoin = WK > 1 ? 4 * 32 * DP * 4 + 4 * 64 * 4 : 0;
  static constexpr int kLds = kLoop > kJoin ? kLoop : kJoin;
};

// The key tiles t0 .. t1 of a workgroup: K and V into the tile buffers, and which keys count.  A tile that is not whole
// (its end, or any tile under a mask) has a bias of 0 or -inf a key in a ring of three: under a mask the lanes that ask
// for a masked row behind the range read it while the tile after next's mask bytes are on their way, so no load waits
// for another (333 masked keys, 44 rows: 25 us unmasked; 36 with the mask read where it is used).
template <class T, int DP, class Sh>
struct KeyStream {
  static constexpr int kKeys = Sh::kKeys;
  KeyTile<T, DP, kKeys> kt, vt;
  const uint8_t* mask;
  float* ring;
  uint32_t lds0;
  int n, t0, t1, tid, slot;   // slot: the ring's entry of the current tile
  float ahead;
  __device__ __forceinline__ void init(const Att& a, int c, int hk, int split, char* lds, int tid_) {
    constexpr int64_t e = (int64_t)sizeof(T);
    tid = tid_;
    lds0 = lds_address(lds);
    ring = reinterpret_cast<float*>(lds + Sh::kBias);
    n = key_count(a, c);
    const int nt = (n + kKeys - 1) / kKeys, share = (nt + a.splits - 1) / a.splits;
    t0 = min(split * share, nt);
    t1 = min(t0 + share, nt);
    mask = a.mask ? a.mask + (int64_t)c * a.Lk : nullptr;
    kt.init(a.k + ((int64_t)c * a.ks[0] + (int64_t)hk * a.ks[2]) * e, a.ks[1] * e, a.D, tid);
    vt.init(a.v + ((int64_t)c * a.vs[0] + (int64_t)hk * a.vs[2]) * e, a.vs[1] * e, a.D, tid);
  }
  __device__ __forceinline__ bool whole(int t) const { return !mask && (t + 1) * kKeys <= n; }
  __device__ __forceinline__ float bias_of(int t) const {
    const int key = t * kKeys + tid;
    return key < n && (!mask || mask[key]) ? 0.f : -kInf;
  }
  __device__ __forceinline__ const float* bias() const { return ring + slot * kKeys; }
  // tile t, the ring's entry `at`, into buffer `buf`
  __device__ __forceinline__ void fetch(int t, int at, int buf) {
    float* b = ring + at * kKeys;
    auto allowed = [&](int row) { return b[row] == 0.f; };
    kt.load(lds0 + buf * Sh::kBuf, t * kKeys, n - t * kKeys, mask != nullptr, allowed);
    vt.load(lds0 + buf * Sh::kBuf + Sh::kTileBytes, t * kKeys, n - t * kKeys, mask != nullptr, allowed);
    if (!mask && !whole(t) && tid < kKeys) b[tid] = bias_of(t);
  }
  __device__ __forceinline__ void start() {
    slot = 0;
    if (t0 >= t1) return;
    if (mask) {
      if (tid < kKeys) {
        ring[tid] = bias_of(t0);
        if (t0 + 1 < t1) ring[kKeys + tid] = bias_of(t0 + 1);
      }
      __syncthreads();
    }
    fetch(t0, 0, 0);
  }
  // around a tile's products: its tile has landed and every wave is done with the one before; the next loads meanwhile
  __device__ __forceinline__ void begin(int t, int cur) {
    dma_wait();
    __syncthreads();
    if (mask && t + 2 < t1 && tid < kKeys) ahead = bias_of(t + 2);
    if (Sh::kBufs == 2 && t + 1 < t1) fetch(t + 1, next(slot), cur ^ 1);
  }
  __device__ __forceinline__ void end(int t) {
    if (mask && t + 2 < t1 && tid < kKeys) ring[next(next(slot)) * kKeys + tid] = ahead;
    if (Sh::kBufs == 1 && t + 1 < t1) {
      __syncthreads();
      fetch(t + 1, next(slot), 0);
    }
    slot = next(slot);
  }
  static __device__ __forceinline__ int next(int s) { return s == 2 ? 0 : s + 1; }
};

template <class T, int HD, int WR, int WK, int KT, int BUFS>
__global__ __launch_bounds__(256) ECNF_WAVES(waves(HD, sizeof(T), 4, 4)) void att_fwd(Att a) {
  constexpr int DP = tile_width(HD);
  typedef FwdShape<T, DP, WR, WK, KT, BUFS> Sh;
  constexpr int kKeys = Sh::kKeys, NS = HD / 16, ND = (HD + 31) / 32, NB = KT / 32, kRows = 32 * WR;
  constexpr int64_t e = (int64_t)sizeof(T);
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int tid = threadIdx.x, l = tid & 63, w = wave_id(), h = l >> 5, wr = WR == 1 ? 0 : w % WR, wk = WK == 1 ? 0 : w / WR;
  int id = xcd_order(blockIdx.x, gridDim.x);
  const int tile = id % a.tiles;
  id /= a.tiles;
  const int split = id % a.splits;
  id /= a.splits;
  const int hk = id % a.Hk, c = id / a.Hk;

  const int r = tile * kRows + wr * 32 + (l & 31);
  const float sc = log2_scale(a.scale);   // a negative scale turns the queries (exact)
  int b = 0, i = 0, g = 0;
  bool live = r < a.R;
  if (live) {
    row_of(a, c, r, b, i, g);
    live = row_live(a, b, i);
  }
  const char* qrow = live ? a.q + ((int64_t)b * a.qs[0] + (int64_t)i * a.qs[1] + (int64_t)(hk * a.G + g) * a.qs[2]) * e : nullptr;
  typename Ops<T>::Frag qf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    qf[s] = frag_global<T>(qrow, s, h, a.D);
    if (a.scale < 0.f) qf[s] = -qf[s];
  }

  KeyStream<T, DP, Sh> ks;
  ks.init(a, c, hk, split, lds, tid);
  Reader<T, DP> rd;
  rd.init(ks.lds0, l);

  f32x16 o[ND];
  float m = -kInf, sum = 0.f;
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f32x16{};
  const bool idle = tile * kRows + wr * 32 >= a.R;
  const float slack = fminf(8.f / sc, 1e38f);   // P may reach 2^8 before the running maximum moves (a rescale of O less often)
  ks.start();
  auto step = [&](int t, auto which) {
    constexpr int cur = decltype(which)::value;
    ks.begin(t, cur);
    const uint32_t kat = cur * Sh::kBuf, vat = kat + Sh::kTileBytes;
    const float* bias = ks.bias();
    if (!idle && (WK == 1 || t * kKeys + wk * KT < ks.n)) {   // the wave has rows, and keys of this tile
      f32x16 sx[NB];
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        sx[kb] = f32x16{};
#pragma unroll
        for (int s = 0; s < NS; ++s) sx[kb] = Ops<T>::mma(rd.frag(kat, wk * KT + kb * 32, s), qf[s], sx[kb]);
      }
      if (!ks.whole(t)) {
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f32x4 bs = *reinterpret_cast<const f32x4*>(bias + wk * KT + kb * 32 + 8 * j + 4 * h);
#pragma unroll
            for (int y = 0; y < 4; ++y) sx[kb][4 * j + y] += bs[y];
          }
      }
      float mx = -kInf;
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int y = 0; y < 16; ++y) mx = fmaxf(mx, sx[kb][y]);
      mx = max_halves(mx);
      if (__any(mx > m + slack)) {
        const float mn = fmaxf(m, mx);
        const float al = __builtin_amdgcn_exp2f((m - (mn == -kInf ? 0.f : mn)) * sc);
        sum *= al;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int y = 0; y < 16; ++y) o[d][y] *= al;
        m = mn;
      }
      const float ref = m == -kInf ? 0.f : -m * sc;   // nothing allowed yet: exp2(-inf) = 0
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int y = 0; y < 16; ++y) {
          sx[kb][y] = __builtin_amdgcn_exp2f(fmaf(sx[kb][y], sc, ref));
          sum += sx[kb][y];
        }
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const auto p = to_frag<T>(sx[kb], s);
#pragma unroll
          for (int d = 0; d < ND; ++d) o[d] = Ops<T>::mma(rd.frag_t(vat, wk * KT + kb * 32 + 16 * s, d), p, o[d]);
        }
    }
    ks.end(t);
  };
  // the buffer is a constant of each half: every LDS address is a register of the loop plus a constant offset
  for (int t = ks.t0; t < ks.t1; t += Sh::kBufs) {
    step(t, Const<0>{});
    if (Sh::kBufs == 2 && t + 1 < ks.t1) step(t + 1, Const<1>{});
  }

  // ---- join the key waves, normalise, store.  lse in log2 units; an empty row has sum 0: output 0, lse -inf
  const int64_t n_rows = (int64_t)a.C * a.Hk * a.R, row0 = ((int64_t)c * a.Hk + hk) * a.R;
  auto put = [&](int rr, bool lv, int bb, int ii, int gg, int d, f32x4 v) {
    if (!lv) v = f32x4{0.f, 0.f, 0.f, 0.f};   // a row behind its molecule's length
    if (a.splits > 1) *reinterpret_cast<f32x4*>(a.part + (split * n_rows + row0 + rr) * a.D + d) = v;
    else store4<T>(a.out + ((((int64_t)bb * a.Lq + ii) * a.Hq + hk * a.G + gg) * a.D + d) * e, v);
  };
  auto put_lse = [&](int rr, bool lv, int bb, int ii, int gg, float mm, float ll) {
    const float lse = ll == 0.f || !lv ? -kInf : mm * sc + __builtin_amdgcn_logf(ll);
    if (a.splits > 1) a.part_lse[split * n_rows + row0 + rr] = lse;
    else if (a.lse) a.lse[((int64_t)bb * a.Hq + hk * a.G + gg) * a.Lq + ii] = lse * kLn2;
  };
  if constexpr (WK == 1) {
    const float tot = sum_halves(sum);
    const float inv = tot > 0.f ? 1.f / tot : (tot == 0.f ? 0.f : tot);   // NaN stays
    if (r < a.R) {
      row_of(a, c, r, b, i, g);
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int dd = 32 * d + 8 * j + 4 * h;
          if (dd < a.D)
            put(r, live, b, i, g, dd,
                f32x4{o[d][4 * j] * inv, o[d][4 * j + 1] * inv, o[d][4 * j + 2] * inv, o[d][4 * j + 3] * inv});
        }
      if (h == 0) put_lse(r, live, b, i, g, m, tot);
    }
  } else {
    float* jo = reinterpret_cast<float*>(lds);                 // [wave][row][DP], 16-byte chunks swizzled by row
    float* jm = jo + 4 * 32 * DP;                              // [wave][row]
    float* jl = jm + 4 * 32;
    const float tot = sum_halves(sum);
    __syncthreads();
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(reinterpret_cast<char*>(jo + w * 32 * DP) + Tile<float, DP>::at(l & 31, 8 * d + 2 * j + h)) =
            f32x4{o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]};
    if (h == 0) jm[w * 32 + (l & 31)] = m, jl[w * 32 + (l & 31)] = tot;
    __syncthreads();
    for (int x = tid; x < WR * 32 * (DP / 4); x += 256) {
      const int ch = x % (DP / 4), row = x / (DP / 4), rw = row >> 5, rl = row & 31;
      const int rr = tile * kRows + row;
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
        const float f = __builtin_amdgcn_exp2f((jm[ww * 32 + rl] - ref) * sc);
        L += f * jl[ww * 32 + rl];
        const f32x4 y = *reinterpret_cast<const f32x4*>(reinterpret_cast<const char*>(jo + ww * 32 * DP) + Tile<float, DP>::at(rl, ch));
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = fmaf(f, y[q], v[q]);
      }
      const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] *= inv;
      int bb, ii, gg;
      row_of(a, c, rr, bb, ii, gg);
      const bool lv = row_live(a, bb, ii);
      put(rr, lv, bb, ii, gg, ch * 4, v);
      if (ch == 0) put_lse(rr, lv, bb, ii, gg, M, L);
    }
  }
}

// joins the splits of the forward pass: out = sum_s 2^(lse_s - M) part_s / sum_s 2^(lse_s - M); a thread has 4 columns.
// Its loads are in flight together (one by one, 64 splits of 32 rows took 20 us of a 151 us call).
template <class T>
__global__ __launch_bounds__(256) void att_fwd_join(Att a) {
  const int64_t n = (int64_t)a.C * a.Hk * a.R;
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int D4 = a.D / 4;
  const int64_t row = x / D4;
  if (row >= n) return;
  const int ch = (int)(x - row * D4);
  float M = -kInf;
#pragma unroll 16
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.part_lse[s * n + row]);
  const float ref = M == -kInf ? 0.f : M;
  float L = 0.f;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 16
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
//
// Bound by the matrix units (busy 0.55 of 1.9 GHz, vector 0.37): 4096 queries of 32 heads on 8192 keys of 8, 128 wide,
// bf16, 745 us, 1107 TFLOP/s of its three products; 22 x 129 in fp32, 2048 times, 20 us, by latency (four short phases a
// workgroup).
// ---------------------------------------------------------------------------------------------------------------
template <class T, int HD, int WR, int WK, int KT, int BUFS>
__global__ __launch_bounds__(256) ECNF_WAVES(waves(HD, sizeof(T), 4, 3)) void att_dq(Att a) {
  constexpr int DP = tile_width(HD);
  typedef FwdShape<T, DP, WR, WK, KT, BUFS> Sh;
  constexpr int kKeys = Sh::kKeys, NS = HD / 16, ND = (HD + 31) / 32, NB = KT / 32;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int tid = threadIdx.x, l = tid & 63, w = wave_id(), h = l >> 5, wr = WR == 1 ? 0 : w % WR, wk = WK == 1 ? 0 : w / WR;
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
  const float sg = a.scale < 0.f ? -1.f : 1.f, sc = sg * log2_scale(a.scale);
  float lse = kInf;
  if (live) {
    lse = a.lse[((int64_t)b * a.Hq + hq) * a.Lq + i] * kLog2e;
    if (lse == -kInf) lse = kInf;
  }
  KeyStream<T, DP, Sh> ks;
  ks.init(a, c, hk, split, lds, tid);
  const uint8_t first = ks.mask && l < ks.n ? ks.mask[l] : (uint8_t)0;
  bool one = false;
  Reader<T, DP> rd;
  rd.init(ks.lds0, l);

  const bool idle = tile * 32 * WR + wr * 32 >= a.R;
  Range<T> range;
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
  const float shift = Range<T>::kShift - lse;
  // P (2^kShift of it) and dP of the 32 keys from k0 of the tile at kat, vat
  auto products = [&](int t, uint32_t kat, uint32_t vat, int k0, f32x16& p, f32x16& dp) __attribute__((always_inline)) {
    p = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      p = Ops<T>::mma(rd.frag(kat, k0, s), qf[s], p);
      dp = Ops<T>::mma(rd.frag(vat, k0, s), df[s], dp);
    }
    if (!ks.whole(t)) {
      if (one) dp *= 0.f;
      const float* bias = ks.bias();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 bs = *reinterpret_cast<const f32x4*>(bias + k0 + 8 * j + 4 * h);
#pragma unroll
        for (int x = 0; x < 4; ++x) p[4 * j + x] = bs[x] < 0.f ? bs[x] * sg : p[4 * j + x];
      }
    }
#pragma unroll
    for (int x = 0; x < 16; ++x) p[x] = __builtin_amdgcn_exp2f(fmaf(p[x], sc, shift));
  };
  ks.start();
  one = one_key(ks.mask, ks.n, l, __ballot(first != 0));   // (behind the start's own wait for mask bytes)
  // A context whose length is one tile: delta = sum_j P dP over its keys instead of sum_d dO O.  With few keys dP - delta
  // cancels, and O was rounded (bf16: dQ and dK of 2-key rows 2.6e-3 off, so 1.7e-3, which is their own rounding); with many,
  // O is an average and its rounding is small beside dP.  (Few keys that a mask leaves of many tiles keep delta from O: to
  // sum over them first would read all tiles twice.)  The scores are made twice: nothing for 16-bit types (fp32's O is exact
  // enough; there it would cost 74 -> 79 us of the 22 x 129 training pass).
  if (sizeof(T) == 2 && ks.t0 < ks.t1 && ks.n <= kKeys) {
    dma_wait();
    __syncthreads();
    float sum = 0.f;
    if (!idle)
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        const int k0 = wk * KT + kb * 32;
        if (k0 >= ks.n) break;
        f32x16 p, dp;
        products(0, 0, Sh::kTileBytes, k0, p, dp);
#pragma unroll
        for (int x = 0; x < 16; ++x) sum = fmaf(p[x], dp[x], sum);
      }
    sum = sum_halves(sum) * Range<T>::kBack;
    if constexpr (WK == 1) {
      delta = sum;
    } else {
      float* part = reinterpret_cast<float*>(lds + Sh::kDelta);
      if (h == 0) part[w * 32 + (l & 31)] = sum;
      __syncthreads();
      delta = 0.f;
#pragma unroll
      for (int k = 0; k < WK; ++k) delta += part[(k * WR + wr) * 32 + (l & 31)];
    }
  }
  if (one) delta *= 0.f;   // with dP: dS is 0 and not what the two differ by
  if (split == 0 && wk == 0 && h == 0 && r < a.R) {
    const int64_t row = ((int64_t)c * a.Hk + hk) * a.R + r;
    a.row_lse[row] = lse;
    a.row_delta[row] = delta;
  }
  auto step = [&](int t, auto which) {
    constexpr int cur = decltype(which)::value;
    ks.begin(t, cur);
    const uint32_t kat = cur * Sh::kBuf, vat = kat + Sh::kTileBytes;
    if (!idle)
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
      const int k0 = wk * KT + kb * 32;
      if (t * kKeys + k0 >= ks.n) break;
      f32x16 sx, dp;
      products(t, kat, vat, k0, sx, dp);
#pragma unroll
      for (int x = 0; x < 16; ++x) sx[x] *= dp[x] - delta;
      range.fit(sx, acc, ND);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const auto dsf = to_frag<T>(sx, s);
        // Narrow heads: dQ is P's covariance of dP and K, and dS's rounding errors meet K with its mean, which is the
        // larger part the narrower the head.  So what was rounded away is added by a second product (16 wide, bf16:
        // dQ's error 2.5e-3 -> 1.8e-3, of which 1.7e-3 its own rounding; gradients of 2000 on 4000 keys 178 -> 208 us,
        // of 22 on 129 keys 34 -> 35).
        constexpr bool rest = sizeof(T) == 2 && HD <= 32;
        typename Ops<T>::Frag lo;
        if constexpr (rest)
#pragma unroll
          for (int x = 0; x < 8; ++x) lo[x] = (T)(sx[8 * s + x] - (float)dsf[x]);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const auto kf = rd.frag_t(kat, k0 + 16 * s, d);
          acc[d] = Ops<T>::mma(kf, dsf, acc[d]);
          if constexpr (rest) acc[d] = Ops<T>::mma(kf, lo, acc[d]);
        }
      }
    }
    ks.end(t);
  };
  // the buffer is a constant of each half: every LDS address is a register of the loop plus a constant offset
  for (int t = ks.t0; t < ks.t1; t += Sh::kBufs) {
    step(t, Const<0>{});
    if (Sh::kBufs == 2 && t + 1 < ks.t1) step(t + 1, Const<1>{});
  }

  if constexpr (Range<T>::kShift != 0.f) {
    const float back = range.back();
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] *= back;
  }
  if (lse == kInf)   // a row without keys: 0, also where its dO is NaN
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
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
//
// Bound by the matrix units and, at 128, by the registers: two gradients of 32 keys take half of them, which leaves two
// waves a SIMD and few reads ahead (MFMA busy 0.45, vector 0.35, LDS 0.34; 2.1 GHz).  4096 queries of 32 heads on 8192
// keys of 8, 128 wide, bf16: 1100 us, 1000 TFLOP/s of its four products; with V in registers too 1425.  22 rows x 129
// keys in fp32, 2048 times: 39 us, by latency; the last of a context's five key blocks has a workgroup of its own.
// ---------------------------------------------------------------------------------------------------------------
template <class T, int DP, int WY, int WX>
struct DkvShape {
  // V of the workgroup's keys: registers (a B operand a wave), or LDS where those would leave none to read ahead with
  static constexpr bool kVLds = DP == 128;
  static constexpr int kVBytes = kVLds ? 32 * WY * DP * (int)sizeof(T) : 0;
  // row blocks a wave takes of a tile: 2 where the registers allow (half the barriers; a tile is whole chunks)
  static constexpr int kXB = DP * (int)sizeof(T) <= 128 ? 2 : 1;
  static constexpr int kRows = 32 * WX * kXB;
  static constexpr int kTileBytes = kRows * DP * (int)sizeof(T);
  static constexpr int kBuf = 2 * kTileBytes;   // Q, dO
  static constexpr int kBufs = 2 * (kBuf + kRows * 8) + kVBytes <= 160 * 1024 ? 2 : 1;
  static constexpr int kV = kBufs * kBuf;       // behind the tiles: V, then the rows' lse and delta
  static constexpr int kStat = kV + kVBytes;
  static constexpr int kLoop = kStat + kBufs * kRows * 8;
  static constexpr int kJoin = WX > 1 ? 4 * 32 * DP * 4 : 0;
  static constexpr int kLds = kLoop > kJoin ? kLoop : kJoin;
};

template <class T, int HD, int WY, int WX>
__global__ __launch_bounds__(256) ECNF_WAVES(waves(HD, sizeof(T), 3, 2)) void att_dkv(Att a) {
  constexpr int DP = tile_width(HD);
  typedef DkvShape<T, DP, WY, WX> Sh;
  constexpr int kRows = Sh::kRows, NS = HD / 16, ND = (HD + 31) / 32;
  constexpr int64_t e = (int64_t)sizeof(T);
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int tid = threadIdx.x, l = tid & 63, w = wave_id(), h = l >> 5, wy = WY == 1 ? 0 : w % WY, wx = WX == 1 ? 0 : w / WY;
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
  // (where one key is left, dP = delta = 0, as in dQ: V, which only dP reads, is taken as 0)
  const uint64_t own = __ballot(ok && l < 32);
  const bool one = own && one_key(mask, n, l, own);
  const char* vrow = ok && !one ? a.v + ((int64_t)c * a.vs[0] + (int64_t)key * a.vs[1] + (int64_t)hk * a.vs[2]) * e : nullptr;
  const uint32_t lds0 = lds_address(lds);
  Reader<T, DP> rdr;
  rdr.init(lds0, l);
  typename Ops<T>::Frag kf[NS], vf[Sh::kVLds ? 1 : NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    kf[s] = frag_global<T>(krow, s, h, a.D);
    const auto x = frag_global<T>(vrow, s, h, a.D);
    if constexpr (Sh::kVLds) {
      // a key's row belongs to the wave that reads it; the row waves (WX) of a key block write the same values
      char* p = lds + Sh::kV;
      const int r = wy * 32 + (l & 31);
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<typename Ops<T>::Frag*>(p + Tile<T, DP>::at(r, 2 * s + h)) = x;
      } else {
        *reinterpret_cast<f32x4*>(p + Tile<T, DP>::at(r, 4 * s + 2 * h)) = f32x4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4*>(p + Tile<T, DP>::at(r, 4 * s + 2 * h + 1)) = f32x4{x[4], x[5], x[6], x[7]};
      }
    } else {
      vf[s] = x;
    }
  }
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dk[d] = f32x16{}, dv[d] = f32x16{};

  // no key of the workgroup is inside its context: nothing to sum (the rows loop is uniform over the workgroup)
  const int nt = tile * WY * 32 < n ? (a.R + kRows - 1) / kRows : 0, share = (nt + a.splits - 1) / a.splits;
  const int t0 = min(split * share, nt), t1 = min(t0 + share, nt);
  const int64_t row0 = ((int64_t)c * a.Hk + hk) * a.R;
  const float sc = copysignf(log2_scale(a.scale), a.scale);

  float* const stats = reinterpret_cast<float*>(lds + Sh::kStat);
  const bool idle = (tile * WY + wy) * 32 >= n;
  Range<T> range;
  const bool fast = a.flat && !a.qlen && kRows % a.G == 0;
  RowTile<T, DP, kRows> tq, td;
  tq.init(a, a.q, a.qs, c, hk, tid, fast);
  td.init(a, a.dout, a.ds, c, hk, tid, fast);
  float nl = kInf, nd = 0.f;
  auto fetch = [&](int t, int buf) {
    const int r0 = t * kRows;
    tq.load(a, lds0 + buf * Sh::kBuf, c, r0, tid, fast);
    td.load(a, lds0 + buf * Sh::kBuf + Sh::kTileBytes, c, r0, tid, fast);
    if (tid < kRows) {
      const bool in = r0 + tid < a.R;
      nl = in ? a.row_lse[row0 + r0 + tid] : kInf;
      nd = in ? a.row_delta[row0 + r0 + tid] : 0.f;
    }
  };
  auto publish = [&](int buf) {
    if (tid < kRows) stats[buf * 2 * kRows + tid] = nl - Range<T>::kShift, stats[(buf * 2 + 1) * kRows + tid] = nd;
  };
  if (t0 < t1) {
    fetch(t0, 0);
    publish(0);
  }
  for (int t = t0; t < t1; ++t) {
    const int cur = Sh::kBufs == 2 ? (t - t0) & 1 : 0, next = Sh::kBufs == 2 ? cur ^ 1 : 0;
    dma_wait();
    __syncthreads();   // tile t has landed, and every wave is done with tile t - 1
    if (Sh::kBufs == 2 && t + 1 < t1) fetch(t + 1, next);
    const uint32_t qat = cur * Sh::kBuf, dat = qat + Sh::kTileBytes;
    const float* rl = stats + cur * 2 * kRows;
    const float* rd = rl + kRows;
    if (!idle)
#pragma unroll
    for (int xb = 0; xb < Sh::kXB; ++xb) {
      const int x0 = (wx * Sh::kXB + xb) * 32;
      if (t * kRows + x0 >= a.R) break;
      f32x16 sx = f32x16{}, dp = f32x16{};
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        sx = Ops<T>::mma(rdr.frag(qat, x0, s), kf[s], sx);
        if constexpr (Sh::kVLds) dp = Ops<T>::mma(rdr.frag(dat, x0, s), rdr.frag(Sh::kV, wy * 32, s), dp);
        else dp = Ops<T>::mma(rdr.frag(dat, x0, s), vf[s], dp);
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
      range.fit(dp, dk, ND);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const auto pf = to_frag<T>(sx, s), sf = to_frag<T>(dp, s);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          dv[d] = Ops<T>::mma(rdr.frag_t(dat, x0 + 16 * s, d), pf, dv[d]);
          dk[d] = Ops<T>::mma(rdr.frag_t(qat, x0 + 16 * s, d), sf, dk[d]);
        }
      }
    }
    if (t + 1 < t1) {
      if (Sh::kBufs == 1) {
        __syncthreads();
        fetch(t + 1, next);
      }
      publish(next);
    }
  }

  if constexpr (Range<T>::kShift != 0.f) {
    const float back = range.back();
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] *= back, dv[d] *= Range<T>::kBack;
  }
  if (!ok)   // a key that no row may read: 0, also where a dO is NaN
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] = dv[d] = f32x16{};
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

// sums the splits' partials (in order): which = 0 dQ rows, 1 dK and dV keys (blockIdx.y: 0 dK, 1 dV); 4 columns a thread.
// 16 splits of 512 keys of 8 x 64 (fp16 gradients): 8 us, most of it start and end.
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
#pragma unroll 16
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
  int narrow;        // 1: the waves split the loop (few rows / few keys), 0: the rows (forward, dQ) or keys (dK dV)
  int single;        // one tile buffer (few tiles: more workgroups fit a CU), else two (the next tile loads meanwhile)
  int tiles, splits;
  int64_t grid, part, part_lse;   // workgroups; workspace floats
};

inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// outer: rows (forward, dQ) or keys (dK dV) of a (context, key head); inner: the loop's length, and its tiles';
// per_row: partial floats of one outer element and split.
//
// The loop is split until the workgroups fill the chip once (one a CU where a row of a tile has 256 bytes or more: their
// buffers fill its LDS; else two), but into parts of no fewer than 2 tiles (narrow), 8 (16-bit types) or 4 (fp32, whose
// tiles take longer).  Both sides measured, us, as it is | the other way:
//   one a CU: one token, 131072 keys of 8 x 128, bf16 111 | two 129; 1000 rows on 4000 keys of 4 x 128, fp32 92 | 115 (but
//     gradients of 256 x 22 rows on 512 shared keys of 8 x 64, fp32 297 | 275)
//   two a CU: one token, 4 x 16384 keys of 8 x 64, bf16 29 | one 31; those gradients in fp16 74 | 77
//   narrow: gradients of 4 rows on 16 x 2048 keys of 2 x 64, fp32 60 | parts of 4 70, of 1 60; bf16 49 | 49, 47
//   16-bit: gradients of 256 x 22 rows on 512 shared keys of 8 x 64, bf16 70 | parts of 4 94, of 16 72; of 100 rows on
//     2 x 4000 keys of 4 x 64, bf16 50 | 50, 71
//   fp32: 100 rows on 2 x 4000 keys of 4 x 64 37 | parts of 8 50, of 2 34; gradients of 300 rows on 2000 keys 98 | 157, 65
// One tile buffer for narrow parts of at most two tiles: fp32 22 x 129 training pass 74 | two 84; two buffers for more: one
// token on 64 x 8192 keys of 8 x 128, bf16 382 | one 410.
inline Plan make_plan(const Att& a, int outer, int inner, int narrow_step, int wide_step, int64_t per_row, bool lse) {
  Plan p;
  const int64_t pairs = (int64_t)a.C * a.Hk;
  p.narrow = outer <= 32;
  p.tiles = ceil_div(outer, p.narrow ? 32 : 128);
  const int64_t base = pairs * p.tiles;
  const int fill = tile_width(a.D) * a.elem > 128 ? 256 : 512, least = p.narrow ? 2 : a.elem == 4 ? 4 : 8;
  const int inner_tiles = ceil_div(inner, p.narrow ? narrow_step : wide_step);
  int64_t s = 1;
  if (base > 0 && base < fill) s = (fill + base - 1) / base;
  if (s > inner_tiles / least) s = inner_tiles / least;
  const int64_t one = pairs * outer * per_row;
  if (one > 0 && s * one > kPartMax) s = kPartMax / one;
  p.splits = (int)(s < 1 ? 1 : s);
  p.single = inner_tiles <= 2 * p.splits;
  p.grid = base * p.splits;
  p.part = p.splits > 1 ? (int64_t)p.splits * one : 0;
  p.part_lse = p.splits > 1 && lse ? (int64_t)p.splits * pairs * outer : 0;
  return p;
}
inline Plan plan_fwd(const Att& a) { return make_plan(a, a.R, a.Lk, 128, 64, a.D, true); }
inline Plan plan_dq(const Att& a) { return make_plan(a, a.R, a.Lk, 128, 64, a.D, false); }
inline Plan plan_dkv(const Att& a) { return make_plan(a, a.Lk, a.R, 128, 32, 2 * a.D, false); }

// one per element type (ecnf_attention.hip)
hipError_t launch_fwd_bf16(const Att&, hipStream_t);
hipError_t launch_fwd_f16(const Att&, hipStream_t);
hipError_t launch_fwd_f32(const Att&, hipStream_t);
hipError_t launch_grad_bf16(const Att&, hipStream_t);
hipError_t launch_grad_f16(const Att&, hipStream_t);
hipError_t launch_grad_f32(const Att&, hipStream_t);

}  // namespace ecnf_ctx
