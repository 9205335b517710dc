// ecnf_attention.hip — launches of the cross attention kernels (context_attention.hpp) for one element type
// (ECNF_ATT_TYPE 0 fp32, 1 bf16, 2 fp16) and direction (ECNF_ATT_GRAD): one translation unit each.
#include "context_attention.hpp"

namespace ecnf_ctx {
namespace {

#if ECNF_ATT_TYPE == 0
typedef float T;
#define ECNF_ATT_NAME(x) x##_f32
#elif ECNF_ATT_TYPE == 1
typedef __bf16 T;
#define ECNF_ATT_NAME(x) x##_bf16
#else
typedef _Float16 T;
#define ECNF_ATT_NAME(x) x##_f16
#endif

template <class K>
hipError_t launch(K kernel, int64_t grid, int lds, const Att& a, hipStream_t s) {
  if (!grid) return hipSuccess;   // no rows or no keys
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
  }
  kernel<<<dim3((unsigned)grid), dim3(256), lds, s>>>(a);
  return hipGetLastError();
}

Att with_plan(Att a, const Plan& p, float* part) {
  a.tiles = p.tiles;
  a.splits = p.splits;
  a.part = part;
  a.part_lse = part + p.part;
  return a;
}

// Few rows (a single token, a small molecule): the waves split the keys, with one tile buffer where a workgroup has at
// most two tiles and two where it has more (make_plan has both measured).  More rows: the waves split the rows and share
// every tile.
#if !ECNF_ATT_GRAD
template <int HD>
hipError_t fwd(const Att& in, hipStream_t s) {
  constexpr int DP = tile_width(HD);
  const Plan p = plan_fwd(in);
  const Att a = with_plan(in, p, in.part);
  hipError_t e = !p.narrow  ? launch(att_fwd<T, HD, 4, 1, 64, 2>, p.grid, FwdShape<T, DP, 4, 1, 64, 2>::kLds, a, s)
                 : p.single ? launch(att_fwd<T, HD, 1, 4, 32, 1>, p.grid, FwdShape<T, DP, 1, 4, 32, 1>::kLds, a, s)
                            : launch(att_fwd<T, HD, 1, 4, 32, 2>, p.grid, FwdShape<T, DP, 1, 4, 32, 2>::kLds, a, s);
  if (e != hipSuccess || p.splits == 1) return e;
  const int64_t n = (int64_t)a.C * a.Hk * a.R * (a.D / 4);
  att_fwd_join<T><<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s>>>(a);
  return hipGetLastError();
}
#else
template <int HD>
hipError_t grad(const Att& in, hipStream_t s) {
  constexpr int DP = tile_width(HD);
  const Plan p = plan_dq(in), y = plan_dkv(in);
  Att a = with_plan(in, p, in.part);
  hipError_t e = !p.narrow  ? launch(att_dq<T, HD, 4, 1, 64, 2>, p.grid, FwdShape<T, DP, 4, 1, 64, 2>::kLds, a, s)
                 : p.single ? launch(att_dq<T, HD, 1, 4, 32, 1>, p.grid, FwdShape<T, DP, 1, 4, 32, 1>::kLds, a, s)
                            : launch(att_dq<T, HD, 1, 4, 32, 2>, p.grid, FwdShape<T, DP, 1, 4, 32, 2>::kLds, a, s);
  if (e != hipSuccess) return e;
  if (p.splits > 1) {
    const int64_t n = (int64_t)a.C * a.Hk * a.R * (a.D / 4);
    att_grad_join<T><<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s>>>(a, 0);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  a = with_plan(in, y, in.part);
  e = y.narrow ? launch(att_dkv<T, HD, 1, 4>, y.grid, DkvShape<T, DP, 1, 4>::kLds, a, s)
               : launch(att_dkv<T, HD, 4, 1>, y.grid, DkvShape<T, DP, 4, 1>::kLds, a, s);
  if (e != hipSuccess || y.splits == 1) return e;
  const int64_t n = (int64_t)a.C * a.Hk * a.Lk * (a.D / 4);
  att_grad_join<T><<<dim3((unsigned)((n + 255) / 256), 2), dim3(256), 0, s>>>(a, 1);
  return hipGetLastError();
}
#endif

}  // namespace

#define ECNF_ATT_BY_WIDTH(f) \
  (a.D <= 16 ? f<16>(a, s) : a.D <= 32 ? f<32>(a, s) : a.D <= 64 ? f<64>(a, s) : a.D <= 96 ? f<96>(a, s) : f<128>(a, s))
#if !ECNF_ATT_GRAD
hipError_t ECNF_ATT_NAME(launch_fwd)(const Att& a, hipStream_t s) { return ECNF_ATT_BY_WIDTH(fwd); }
#else
hipError_t ECNF_ATT_NAME(launch_grad)(const Att& a, hipStream_t s) { return ECNF_ATT_BY_WIDTH(grad); }
#endif

}  // namespace ecnf_ctx
