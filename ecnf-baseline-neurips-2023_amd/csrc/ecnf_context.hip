// ecnf_context.hip — the context operators of include/ecnf.h: per-head norm and rotation of queries and keys (kernels
// here), and the host side of cross attention (kernels: context_attention.hpp, one unit per element type).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>

#include "../../include/ecnf.h"
#include "context_attention.hpp"

namespace ecnf {
int set_error(int code, const char* msg);   // ecnf_hip.hip
}

namespace ecnf_ctx {
namespace {

// ---------------------------------------------------------------------------------------------------------------
// norm + rotation.  For every (token, head) row x of D elements:
//   y = w x r,  r = 1 / sqrt(mean(x^2) + eps);  pair j of axis a turns by p_a theta^(-2j / d_a):
//   (lo, hi) -> (lo c - hi s, lo s + hi c);  dims behind the axes pass through (a pair whose angle is 0).
// backward: g = the turned-back gradient, u = w g,  dx = r (u - x r^2 mean(u x)),  dw = sum over rows of g x r.
//
// Memory bound (each element read once, written once).  A workgroup takes tiles of a few tokens: their sines and
// cosines are computed once (fp64 product and reduction to a quarter turn, so far positions keep their angle; then
// fp32) into LDS, and every head of the token uses them from there.  A row is VE pairs a lane on LP lanes; a lane loads
// its pairs' two halves (or 2 VE neighbours when interleaved) as up to 16-byte accesses.
//
// Measured, bf16, 128 wide: 4 x 4096 queries of 32 heads and 4 x 8192 keys of 8 on three axes 84 us, 4.8 TB/s (a copy:
// 5.2 to 5.5); the backward pass of 4 x 4095 and 4 x 2047 90 us, 5.0 TB/s, and 8 us for the weights.  With the loads
// behind the angles instead of before them the first took 97 us.  Small calls (1024 x 13 atoms, fp32) are one launch
// of 7 us, nearly all of it its start and end.
// ---------------------------------------------------------------------------------------------------------------
constexpr int kMaxPairs = 64;
constexpr int kCsEntries = 2048;   // (cos, sin) of a tile: 16 KiB of LDS
constexpr int kMaxGradBlocks = 1024;

struct NormSide {
  const char *x, *dy;
  char* out;
  const float* w;
  float* dw;
  const char* pos;
  int64_t xs[3], gs[3], ps[2];
  int32_t tokens, L, H, pos_type, tt, tiles, blocks;   // tt: tokens of a tile
  FastDiv dL, dH;
};
struct Norm {
  NormSide s[2];   // q, k
  float* part;     // backward: [block][D] weight gradient partials, q's blocks first
  int32_t D, half, lp, n_axes, interleaved;
  float eps;
  int32_t first[5];   // first pair of each axis; the entry behind the last axis: first pair without rotation
  double turns[kMaxPairs];   // theta^(-2j/d) / (2 pi)
};

__device__ __forceinline__ double position(const NormSide& s, const char* p) {
  if (s.pos_type == ECNF_POS_I32) return (double)*reinterpret_cast<const int32_t*>(p);
  if (s.pos_type == ECNF_POS_I64) return (double)*reinterpret_cast<const int64_t*>(p);
  return (double)*reinterpret_cast<const float*>(p);
}

// cos and sin of 2 pi t: quarter turns off in fp64, the rest (|angle| <= pi / 4) in fp32
__device__ __forceinline__ float2 cos_sin(double t) {
  const double u = 4.0 * (t - rint(t)), n = rint(u);
  float s, c;
  sincospif(0.5f * (float)(u - n), &s, &c);
  const int k = (int)n & 3;
  const float a = (k & 1) ? s : c, b = (k & 1) ? c : s;
  return make_float2((k == 1 || k == 2) ? -a : a, (k & 2) ? -b : b);
}

// a lane's VE pairs of a row as loaded: [lo .., hi ..], or 2 VE neighbours (interleaved)
template <class T, int VE, bool inter>
struct Pairs {
  typedef T V __attribute__((ext_vector_type(VE)));
  V u, v;
  __device__ __forceinline__ void load(const char* row, int lo, int hi) {
    u = *reinterpret_cast<const V*>(row + lo * (int)sizeof(T));
    v = *reinterpret_cast<const V*>(row + (inter ? lo + VE : hi) * (int)sizeof(T));
  }
  __device__ __forceinline__ void store(char* row, int lo, int hi) const {
    *reinterpret_cast<V*>(row + lo * (int)sizeof(T)) = u;
    *reinterpret_cast<V*>(row + (inter ? lo + VE : hi) * (int)sizeof(T)) = v;
  }
  __device__ __forceinline__ void get(float* a, float* b) const {
#pragma unroll
    for (int i = 0; i < VE; ++i) a[i] = (float)at(inter ? 2 * i : i), b[i] = (float)at(inter ? 2 * i + 1 : VE + i);
  }
  __device__ __forceinline__ void set(const float* a, const float* b) {
    T w[2 * VE];
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (inter) w[2 * i] = (T)a[i], w[2 * i + 1] = (T)b[i];
      else w[i] = (T)a[i], w[VE + i] = (T)b[i];
#pragma unroll
    for (int i = 0; i < VE; ++i) u[i] = w[i], v[i] = w[VE + i];
  }
  __device__ __forceinline__ T at(int i) const { return i < VE ? u[i] : v[i - VE]; }
};

__device__ __forceinline__ int axis_of(const Norm& a, int pair) {   // n_axes: not rotated
  int x = 0;
  while (x < a.n_axes && pair >= a.first[x + 1]) ++x;
  return x;
}

template <class T, int VE, bool inter, bool GRAD>
__global__ __launch_bounds__(256) void qk_norm_kernel(Norm a) {
  constexpr int U = GRAD ? 1 : 2;   // (two in the backward pass: 104 us of 96 at 453 MB, its registers cost a wave of four)
  __shared__ float2 cs[kCsEntries];
  __shared__ float red[GRAD ? 256 * 2 * VE : 1];
  const int tid = threadIdx.x;
  const bool second = (int)blockIdx.x >= a.s[0].blocks;
  const NormSide& s = a.s[second];
  const int block = (int)blockIdx.x - (second ? a.s[0].blocks : 0);
  const int ln = tid & (a.lp - 1), slot = tid / a.lp, slots = 256 / a.lp;
  const int p0 = ln * VE;
  const bool on = p0 < a.half;
  int lo = 2 * p0, hi = lo;
  if (!inter && on) {
    const int x = axis_of(a, p0), f0 = x ? a.first[x] : 0, n = (x < a.n_axes ? a.first[x + 1] : a.half) - f0;
    lo = f0 + p0;   // 2 f0 + (p0 - f0)
    hi = lo + n;
  }
  float wa[VE], wb[VE], ga[VE], gb[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    const int e = inter ? lo + 2 * i : lo + i, f = inter ? e + 1 : hi + i;
    wa[i] = s.w && on ? s.w[e] : 1.f;
    wb[i] = s.w && on ? s.w[f] : 1.f;
    ga[i] = gb[i] = 0.f;
  }
  for (int tile = block; tile < s.tiles; tile += s.blocks) {
    const int tok0 = tile * s.tt, nt = min(s.tt, s.tokens - tok0), rows = nt * s.H;
    // U rows at once: their loads are in flight together, the first ones while the angles are made
    Pairs<T, VE, inter> px[U], pd[GRAD ? U : 1];
    int tt[U], head[U];
    auto fetch = [&](int rs) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int rr = min(rs + u * slots, rows - 1);   // behind the last row: read again, not written
        tt[u] = (int)s.dH.div(rr);
        head[u] = rr - tt[u] * s.H;
        const int tok = tok0 + tt[u], b = (int)s.dL.div(tok), i = tok - b * s.L;
        if (on) {
          px[u].load(s.x + ((int64_t)b * s.xs[0] + (int64_t)i * s.xs[1] + (int64_t)head[u] * s.xs[2]) * (int64_t)sizeof(T), lo, hi);
          if constexpr (GRAD)
            pd[u].load(s.dy + ((int64_t)b * s.gs[0] + (int64_t)i * s.gs[1] + (int64_t)head[u] * s.gs[2]) * (int64_t)sizeof(T), lo, hi);
        }
      }
    };
    fetch(slot);
    if (GRAD) __syncthreads();
    for (int x = tid; x < nt * a.half; x += 256) {
      const int t = x / a.half, p = x - t * a.half;
      const int ax = axis_of(a, p);
      float2 v = make_float2(1.f, 0.f);
      if (ax < a.n_axes) {
        const int tok = tok0 + t, b = (int)s.dL.div(tok), i = tok - b * s.L;
        const char* pp = s.pos + ((int64_t)b * s.ps[0] + (int64_t)i * s.ps[1] + ax) * (s.pos_type == ECNF_POS_I64 ? 8 : 4);
        v = cos_sin(position(s, pp) * a.turns[p]);
      }
      cs[x] = v;
    }
    __syncthreads();
    for (int rs = slot; rs < rows; rs += U * slots) {
      if (rs != slot) fetch(rs);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float2 t[VE];
#pragma unroll
        for (int q = 0; q < VE; ++q) t[q] = on ? cs[tt[u] * a.half + p0 + q] : make_float2(1.f, 0.f);
        float xa[VE], xb[VE], ya[VE], yb[VE], ss = 0.f, dot = 0.f;
        px[u].get(xa, xb);
        if constexpr (GRAD) {
          float da[VE], db[VE];
          pd[u].get(da, db);
#pragma unroll
          for (int q = 0; q < VE; ++q) {
            ya[q] = fmaf(da[q], t[q].x, db[q] * t[q].y);
            yb[q] = fmaf(db[q], t[q].x, -(da[q] * t[q].y));
            dot = fmaf(ya[q] * wa[q], xa[q], fmaf(yb[q] * wb[q], xb[q], dot));
          }
        }
#pragma unroll
        for (int q = 0; q < VE; ++q) ss = fmaf(xa[q], xa[q], fmaf(xb[q], xb[q], ss));
        if (!on) ss = dot = 0.f;   // lanes beside the row hold nothing
        for (int m = a.lp >> 1; m; m >>= 1) {
          ss += __shfl_xor(ss, m);
          if (GRAD) dot += __shfl_xor(dot, m);
        }
        const float r = 1.f / sqrtf(ss / (float)a.D + a.eps);
        if (!on || rs + u * slots >= rows) continue;
        char* o = s.out + ((int64_t)(tok0 + tt[u]) * s.H + head[u]) * a.D * (int64_t)sizeof(T);
        if constexpr (GRAD) {
          const float m = r * r * (dot / (float)a.D);
#pragma unroll
          for (int q = 0; q < VE; ++q) {
            ga[q] = fmaf(ya[q], xa[q] * r, ga[q]);
            gb[q] = fmaf(yb[q], xb[q] * r, gb[q]);
            ya[q] = r * (ya[q] * wa[q] - xa[q] * m);
            yb[q] = r * (yb[q] * wb[q] - xb[q] * m);
          }
        } else {
#pragma unroll
          for (int q = 0; q < VE; ++q) {
            const float x = xa[q] * r * wa[q], y = xb[q] * r * wb[q];
            ya[q] = fmaf(x, t[q].x, -(y * t[q].y));
            yb[q] = fmaf(x, t[q].y, y * t[q].x);
          }
        }
        Pairs<T, VE, inter> out;
        out.set(ya, yb);
        out.store(o, lo, hi);
      }
    }
  }
  if constexpr (GRAD) {
    if (!s.dw) return;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < VE; ++q) red[tid * 2 * VE + 2 * q] = ga[q], red[tid * 2 * VE + 2 * q + 1] = gb[q];
    __syncthreads();
    // thread ln (< lp) of slot 0's pairs, one element a thread: sum over the slots in order
    for (int x = tid; x < a.lp * 2 * VE; x += 256) {
      const int l2 = x / (2 * VE), q = x - l2 * 2 * VE, pr = l2 * VE + (q >> 1);
      if (pr >= a.half) continue;
      float v = 0.f;
      for (int y = 0; y < slots; ++y) v += red[(y * a.lp + l2) * 2 * VE + q];
      int e = 2 * pr + (q & 1);
      if (!inter) {
        const int ax = axis_of(a, pr), f0 = ax ? a.first[ax] : 0, n = (ax < a.n_axes ? a.first[ax + 1] : a.half) - f0;
        e = f0 + pr + (q & 1) * n;
      }
      a.part[(int64_t)blockIdx.x * a.D + e] = v;
    }
  }
}

// weight gradients: the blocks' partials summed in a fixed order; blockIdx.y: 0 q, 1 k; 16 columns x 64 lanes a block,
// so that a lane's few loads are in flight together (1024 blocks of 128: 8 us; one column a lane over all blocks: 18)
__global__ __launch_bounds__(1024) void qk_norm_dw_kernel(Norm a) {
  __shared__ float red[64][17];
  const NormSide& s = a.s[blockIdx.y];
  if (!s.dw) return;
  const int x = threadIdx.x & 15, d = blockIdx.x * 16 + x, y = threadIdx.x >> 4;
  const float* p = a.part + (blockIdx.y ? (int64_t)a.s[0].blocks * a.D : 0);
  float v = 0.f;
  if (d < a.D) {
#pragma unroll
    for (int k = 0; k < kMaxGradBlocks / 64; ++k) {
      const int b = y + 64 * k;
      if (b < s.blocks) v += p[(int64_t)b * a.D + d];
    }
  }
  red[y][x] = v;
  __syncthreads();
  if (y < 4) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += red[16 * y + k][x];
    red[16 * y][x] = t;   // row 16 y is this lane's own
  }
  __syncthreads();
  if (y == 0 && d < a.D) s.dw[d] = (red[0][x] + red[16][x]) + (red[32][x] + red[48][x]);
}

// ---------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------
int fail(int code, const char* msg) { return ecnf::set_error(code, msg); }

FastDiv fast_div(uint32_t d) {
  FastDiv f;
  f.d = d;
  f.s = 0;
  while ((1ull << f.s) < d) ++f.s;
  f.m = (uint32_t)(((1ull << 32) * ((1ull << f.s) - d)) / d + 1);
  return f;
}

// the operands' device is made current for the launches and the caller's restored afterwards
struct DeviceScope {
  int prev = -1, dev;
  hipError_t err;
  explicit DeviceScope(int d) : dev(d) {
    err = hipGetDevice(&prev);
    if (err == hipSuccess && prev != d) err = hipSetDevice(d);
  }
  ~DeviceScope() {
    if (err == hipSuccess && prev != dev) (void)hipSetDevice(prev);
  }
};

int hip_fail(hipError_t e) {
  char buf[160];
  snprintf(buf, sizeof buf, "HIP: %s", hipGetErrorString(e));
  return fail(ECNF_E_HIP, buf);
}

int elem_size(int dtype) { return dtype == ECNF_DTYPE_F32 ? 4 : 2; }

constexpr int64_t kMaxRows = (1ll << 31) - 1024;   // 32-bit row indices, with room for the last tile
constexpr int64_t kMaxGrid = 1ll << 24;            // a launch has fewer than 2^32 threads, a workgroup 256

bool aligned(const void* p, const int64_t* st, int n, int elem, int bytes) {
  if ((uintptr_t)p % bytes) return false;
  for (int i = 0; i < n; ++i)
    if (st[i] * elem % bytes) return false;
  return true;
}

int build_norm(const ecnf_qk_norm* o, bool grad, Norm* a, int* ve, bool pointers) {
  if (!o) return fail(ECNF_E_INVALID, "NULL argument");
  if (o->dtype < ECNF_DTYPE_F32 || o->dtype > ECNF_DTYPE_F16) return fail(ECNF_E_INVALID, "unknown dtype");
  if (o->head_dim < 2 || o->head_dim > 2 * kMaxPairs || o->head_dim % 2)
    return fail(ECNF_E_UNSUPPORTED, "head_dim must be even and in [2, 128]");
  if (o->n_axes < 1 || o->n_axes > 4) return fail(ECNF_E_INVALID, "1 to 4 rotation axes");
  if (!(o->theta > 0.0) || !std::isfinite(o->theta)) return fail(ECNF_E_INVALID, "theta must be positive");
  if (!(o->eps >= 0.f) || !std::isfinite(o->eps)) return fail(ECNF_E_INVALID, "eps must be >= 0");
  std::memset(a, 0, sizeof *a);
  a->D = o->head_dim;
  a->half = o->head_dim / 2;
  a->n_axes = o->n_axes;
  a->interleaved = o->interleaved != 0;
  a->eps = o->eps;
  const int elem = elem_size(o->dtype);
  // pairs a lane: as many as one 16-byte access holds, if every axis (and the rest) is whole chunks of them
  int v = 16 / elem;
  int at = 0;
  for (int x = 0; x < o->n_axes; ++x) {
    const int d = o->axes[x];
    if (d < 2 || d % 2 || at + d / 2 > a->half) return fail(ECNF_E_INVALID, "axes must be even, >= 2 and sum to at most head_dim");
    // theta^(-2j/d) as powers of theta^(-2/d): in extended precision their error stays below a step of a double
    const long double ratio = std::pow((long double)o->theta, -2.0L / d);
    long double power = 1.0L / 6.283185307179586476925286766559L;
    for (int j = 0; j < d / 2; ++j, power *= ratio) a->turns[at + j] = (double)power;
    while (!a->interleaved && d / 2 % v) v >>= 1;
    at += d / 2;
    a->first[x + 1] = at;
  }
  while (a->half % v || (!a->interleaved && (a->half - at) % v)) v >>= 1;
  const ecnf_qk_side* sides[2] = {&o->q, &o->k};
  for (int k = 0; k < 2; ++k) {
    const ecnf_qk_side& i = *sides[k];
    NormSide& s = a->s[k];
    if (i.batch < 0 || i.length < 0 || i.heads < 0) return fail(ECNF_E_INVALID, "negative size");
    const int64_t tokens = (int64_t)i.batch * i.length;
    if (tokens >= kMaxRows || tokens * (i.heads ? i.heads : 1) >= (1ll << 40) || i.heads > (1 << 20))
      return fail(ECNF_E_UNSUPPORTED, "too many tokens or heads");
    s.tokens = i.heads ? (int32_t)tokens : 0;
    if (!s.tokens) {
      s.dw = i.weight ? i.weight_grad : nullptr;   // no rows: the gradient is 0 (no blocks to sum)
      continue;
    }
    if (pointers && (!i.x || !i.out || !i.positions || (grad && (!i.grad || (i.weight && !i.weight_grad)))))
      return fail(ECNF_E_INVALID, "NULL argument");
    if (i.position_type < ECNF_POS_I32 || i.position_type > ECNF_POS_F32) return fail(ECNF_E_INVALID, "unknown position type");
    s.x = (const char*)i.x;
    s.dy = (const char*)i.grad;
    s.out = (char*)i.out;
    s.w = i.weight;
    s.dw = grad && i.weight ? i.weight_grad : nullptr;
    s.pos = (const char*)i.positions;
    for (int d = 0; d < 3; ++d) s.xs[d] = i.x_stride[d], s.gs[d] = i.grad_stride[d];
    for (int d = 0; d < 2; ++d) s.ps[d] = i.position_stride[d];
    s.L = i.length;
    s.H = i.heads;
    s.pos_type = i.position_type;
    s.dL = fast_div((uint32_t)i.length);
    s.dH = fast_div((uint32_t)i.heads);
    while (v > 1 && (!aligned(s.x, s.xs, 3, elem, v * elem) || !aligned(s.out, nullptr, 0, elem, v * elem) ||
                     (grad && !aligned(s.dy, s.gs, 3, elem, v * elem))))
      v >>= 1;
  }
  *ve = v;
  a->lp = 1;
  while (a->lp * v < a->half) a->lp *= 2;   // <= 64
  for (int k = 0; k < 2; ++k) {
    NormSide& s = a->s[k];
    if (!s.tokens) continue;
    // tokens of a tile: about 4 rows a lane group, unless that leaves fewer than 1024 tiles (then fewer, but a row for
    // every lane group); their angles fit the LDS
    const int64_t want = (4 * 256 / a->lp + s.H - 1) / s.H, few = (s.tokens + 1023) / 1024, one = (256 / a->lp + s.H - 1) / s.H;
    int64_t tt = want < few ? want : few < one ? one : few;
    if (tt > kCsEntries / a->half) tt = kCsEntries / a->half;
    while (tt > 1 && tt * s.H > (1 << 24)) --tt;
    s.tt = (int)(tt < 1 ? 1 : tt);
    s.tiles = ceil_div(s.tokens, s.tt);
    s.blocks = grad && s.tiles > kMaxGradBlocks ? kMaxGradBlocks : s.tiles;
  }
  return ECNF_OK;
}

template <class T, bool GRAD, int VE>
void launch_norm(const Norm& a, unsigned grid, hipStream_t s) {
  if (a.interleaved) qk_norm_kernel<T, VE, true, GRAD><<<grid, 256, 0, s>>>(a);
  else qk_norm_kernel<T, VE, false, GRAD><<<grid, 256, 0, s>>>(a);
}
template <class T, bool GRAD>
void launch_norm(const Norm& a, int ve, unsigned grid, hipStream_t s) {
  if (ve == 8) {
    if constexpr (sizeof(T) == 2) launch_norm<T, GRAD, 8>(a, grid, s);
  } else if (ve == 4) launch_norm<T, GRAD, 4>(a, grid, s);
  else if (ve == 2) launch_norm<T, GRAD, 2>(a, grid, s);
  else launch_norm<T, GRAD, 1>(a, grid, s);
}

// bytes of the backward pass's partials.  The blocks also depend on the operands' alignment: the most there can be
size_t norm_bytes(const Norm& a) {
  size_t blocks = 0;
  for (const NormSide& s : a.s) blocks += s.tokens < kMaxGradBlocks ? s.tokens : kMaxGradBlocks;
  return blocks * a.D * 4;
}

template <bool GRAD>
int run_norm(const ecnf_qk_norm* o, void* ws, size_t bytes, void* stream) {
  Norm a;
  int ve;
  if (int rc = build_norm(o, GRAD, &a, &ve, true)) return rc;
  const int64_t grid = (int64_t)a.s[0].blocks + a.s[1].blocks;
  const bool dw = a.s[0].dw || a.s[1].dw;
  if (GRAD && dw) {
    if (bytes < norm_bytes(a) || (grid && !ws)) return fail(ECNF_E_INVALID, "workspace below ecnf_qk_norm_workspace_size");
    a.part = (float*)ws;
  }
  if (!grid && !(GRAD && dw)) return ECNF_OK;
  if (grid >= kMaxGrid) return fail(ECNF_E_UNSUPPORTED, "too many tokens");
  DeviceScope dev(o->device);
  if (dev.err != hipSuccess) return hip_fail(dev.err);
  const hipStream_t s = (hipStream_t)stream;
  if (grid) {
    if (o->dtype == ECNF_DTYPE_F32) launch_norm<float, GRAD>(a, ve, (unsigned)grid, s);
    else if (o->dtype == ECNF_DTYPE_BF16) launch_norm<__bf16, GRAD>(a, ve, (unsigned)grid, s);
    else launch_norm<_Float16, GRAD>(a, ve, (unsigned)grid, s);
  }
  if (GRAD && dw) qk_norm_dw_kernel<<<dim3((a.D + 15) / 16, 2), 1024, 0, s>>>(a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? ECNF_OK : hip_fail(e);
}

// what: 0 forward, 1 backward
int build_att(const ecnf_attention* o, int what, Att* a, bool pointers) {
  if (!o) return fail(ECNF_E_INVALID, "NULL argument");
  if (o->dtype < ECNF_DTYPE_F32 || o->dtype > ECNF_DTYPE_F16) return fail(ECNF_E_INVALID, "unknown dtype");
  if (o->batch < 0 || o->n_queries < 0 || o->context_length < 0) return fail(ECNF_E_INVALID, "negative size");
  if (o->context_batch < 1 || (o->context_batch != 1 && o->context_batch != o->batch))
    return fail(ECNF_E_INVALID, "context_batch must be 1 or batch");
  if (o->kv_heads < 1 || o->heads < 1 || o->heads % o->kv_heads) return fail(ECNF_E_INVALID, "heads must be a multiple of kv_heads");
  if (o->head_dim < 8 || o->head_dim > 128 || o->head_dim % 8)
    return fail(ECNF_E_UNSUPPORTED, "head_dim must be a multiple of 8 in [8, 128]");
  if (!std::isfinite(o->scale)) return fail(ECNF_E_INVALID, "scale must be finite");
  const int64_t per = o->batch / o->context_batch, G = o->heads / o->kv_heads;
  const int64_t tokens = per * o->n_queries, pairs = (int64_t)o->context_batch * o->kv_heads;
  if (tokens >= kMaxRows || tokens * G >= kMaxRows || o->context_length >= kMaxRows || pairs >= (1ll << 31))
    return fail(ECNF_E_UNSUPPORTED, "too many rows");
  std::memset(a, 0, sizeof *a);
  a->B = o->batch, a->C = o->context_batch, a->Lq = o->n_queries, a->Lk = o->context_length;
  a->Hq = o->heads, a->Hk = o->kv_heads, a->D = o->head_dim, a->G = (int)G;
  a->per = (int)per;
  a->R = (int)(tokens * G);
  a->scale = o->scale;
  a->q = (const char*)o->q, a->k = (const char*)o->k, a->v = (const char*)o->v, a->dout = (const char*)o->out_grad;
  a->out = (char*)o->out, a->dq = (char*)o->q_grad, a->dk = (char*)o->k_grad, a->dv = (char*)o->v_grad;
  a->lse = o->lse;
  a->qlen = o->query_lengths, a->klen = o->context_lengths, a->mask = o->context_mask;
  for (int d = 0; d < 3; ++d)
    a->qs[d] = o->q_stride[d], a->ks[d] = o->k_stride[d], a->vs[d] = o->v_stride[d], a->ds[d] = o->out_grad_stride[d];
  a->dG = fast_div((uint32_t)G);
  a->dL = fast_div((uint32_t)(o->n_queries ? o->n_queries : 1));
  const int e = elem_size(o->dtype);
  a->elem = e;
  for (const int64_t* st : {o->q_stride, o->k_stride, o->v_stride, what ? o->out_grad_stride : o->q_stride})
    for (int d = 0; d < 3; ++d)
      if (st[d] < 0) return fail(ECNF_E_INVALID, "negative stride");
  // tiles of keys are addressed with 32-bit offsets from their first row, tiles of query rows (at most 256) too where
  // the tokens of a context are evenly spaced
  auto span = [&](const int64_t* st, int d) { return st[d] * e * 256 < (1ll << 31); };
  if (o->context_length > 1 && (!span(o->k_stride, 1) || !span(o->v_stride, 1)))
    return fail(ECNF_E_UNSUPPORTED, "rows of k and v must be less than 8 MiB apart");
  // what lies behind the last key reads as zero because it lies behind the last row's end: rows must not overlap
  if (o->context_length > 1 && (o->k_stride[1] < o->head_dim || o->v_stride[1] < o->head_dim))
    return fail(ECNF_E_INVALID, "rows of k and v must not overlap");
  if (o->context_length == 1) a->ks[1] = a->vs[1] = o->head_dim;   // (one row: its stride may be anything)
  auto even = [&](const int64_t* st) {
    return (per <= 1 || o->n_queries <= 1 || st[0] == st[1] * o->n_queries) && span(st, 1) && span(st, 2);
  };
  if (o->n_queries == 1) a->qs[1] = a->qs[0], a->ds[1] = a->ds[0];   // one token a molecule: its stride is the batch's
  a->flat = even(a->qs) && (!what || even(a->ds));
  if (!pointers) return ECNF_OK;
  const bool rows = a->R > 0, keys = a->Lk > 0;
  if ((rows && (!o->q || !o->out)) || (keys && (!o->k || !o->v))) return fail(ECNF_E_INVALID, "NULL argument");
  if (what && ((rows && (!o->out_grad || !o->q_grad || !o->lse)) || (keys && (!o->k_grad || !o->v_grad))))
    return fail(ECNF_E_INVALID, "NULL argument");
  if (!aligned(o->q, o->q_stride, 3, e, 16) || !aligned(o->k, o->k_stride, 3, e, 16) || !aligned(o->v, o->v_stride, 3, e, 16) ||
      !aligned(o->out, nullptr, 0, e, 16) ||
      (what && (!aligned(o->out_grad, o->out_grad_stride, 3, e, 16) || !aligned(o->q_grad, nullptr, 0, e, 16) ||
                !aligned(o->k_grad, nullptr, 0, e, 16) || !aligned(o->v_grad, nullptr, 0, e, 16))))
    return fail(ECNF_E_INVALID, "operands must start rows on 16-byte boundaries");
  return ECNF_OK;
}

size_t align4(size_t floats) { return (floats + 3) / 4 * 4; }

// workspace floats: the splits' partials (one kernel's at a time), in the backward pass behind every row's lse and delta
size_t att_rows(const Att& a) { return align4((size_t)a.C * a.Hk * a.R); }
size_t att_floats(const Att& a, int what) {
  if (!what) {
    const Plan p = plan_fwd(a);
    return p.part + p.part_lse;
  }
  const Plan p = plan_dq(a), y = plan_dkv(a);
  return 2 * att_rows(a) + (size_t)(p.part > y.part ? p.part : y.part);
}

int run_att(const ecnf_attention* o, int what, void* ws, size_t bytes, void* stream) {
  Att a;
  if (int rc = build_att(o, what, &a, true)) return rc;
  if (a.R == 0 && (!what || a.Lk == 0)) return ECNF_OK;
  const size_t need = att_floats(a, what) * 4;
  if (need && (!ws || bytes < need || (uintptr_t)ws % 16))
    return fail(ECNF_E_INVALID, "workspace below ecnf_cross_attention_workspace_size (or not 16-byte aligned)");
  // (the joins' grids are smaller: what they read, splits times their outputs, is at most kPartMax floats)
  if (what ? plan_dq(a).grid >= kMaxGrid || plan_dkv(a).grid >= kMaxGrid : plan_fwd(a).grid >= kMaxGrid)
    return fail(ECNF_E_UNSUPPORTED, "too many rows");
  DeviceScope dev(o->device);
  if (dev.err != hipSuccess) return hip_fail(dev.err);
  const hipStream_t s = (hipStream_t)stream;
  a.part = (float*)ws;
  hipError_t e;
  if (!what) {
    e = o->dtype == ECNF_DTYPE_F32 ? launch_fwd_f32(a, s) : o->dtype == ECNF_DTYPE_BF16 ? launch_fwd_bf16(a, s) : launch_fwd_f16(a, s);
  } else {
    a.row_lse = a.part;
    a.row_delta = a.part + att_rows(a);
    a.part += 2 * att_rows(a);
    e = o->dtype == ECNF_DTYPE_F32 ? launch_grad_f32(a, s) : o->dtype == ECNF_DTYPE_BF16 ? launch_grad_bf16(a, s) : launch_grad_f16(a, s);
  }
  return e == hipSuccess ? ECNF_OK : hip_fail(e);
}

}  // namespace
}  // namespace ecnf_ctx

using namespace ecnf_ctx;

extern "C" {

int ecnf_qk_norm_workspace_size(const ecnf_qk_norm* o, size_t* bytes) {
  if (!bytes) return fail(ECNF_E_INVALID, "NULL argument");
  Norm a;
  int ve;
  if (int rc = build_norm(o, true, &a, &ve, false)) return rc;
  *bytes = norm_bytes(a);
  return ECNF_OK;
}

int ecnf_qk_norm_rotary(const ecnf_qk_norm* o, void* stream) { return run_norm<false>(o, nullptr, 0, stream); }

int ecnf_qk_norm_rotary_grad(const ecnf_qk_norm* o, void* workspace, size_t workspace_bytes, void* stream) {
  return run_norm<true>(o, workspace, workspace_bytes, stream);
}

int ecnf_cross_attention_workspace_size(const ecnf_attention* o, int32_t grad, size_t* bytes) {
  if (!bytes) return fail(ECNF_E_INVALID, "NULL argument");
  Att a;
  if (int rc = build_att(o, grad, &a, false)) return rc;
  *bytes = a.R == 0 && (!grad || a.Lk == 0) ? 0 : att_floats(a, grad) * 4;
  return ECNF_OK;
}

int ecnf_cross_attention(const ecnf_attention* o, void* workspace, size_t workspace_bytes, void* stream) {
  return run_att(o, 0, workspace, workspace_bytes, stream);
}

int ecnf_cross_attention_grad(const ecnf_attention* o, void* workspace, size_t workspace_bytes, void* stream) {
  return run_att(o, 1, workspace, workspace_bytes, stream);
}

}  // extern "C"
