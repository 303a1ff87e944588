// What stands between two blocks of a layer, in one pass over the rows:
//   u = x                                   the block's output
//   u = u / sqrt(mean u^2 + eps) * after    the norm behind the block (optional)
//   h = residual + scale * gate * u         its gate (optional) and residual scale
//   y = h / sqrt(mean h^2 + eps) * before   the norm before the next block (optional)
// h goes out in the residual stream's type, y in x's, or as e4m3 codes with one
// scale for every `group` elements (the formulas of sgl_act_quant, on the fp32 y: no
// rounding to 16 bits lies between).  Everything is fp32 up to the one rounding of each
// output; y is of the h in registers, not of the rounded one.
//
// Bound by HBM: every input is read once and every output written once.  A workgroup
// takes a row, 8 elements a thread and unit in registers across both sums, and goes on
// with the row that lies a grid's length behind, whose loads are on their way during
// the sums; the weights and a gate of channels stay in registers.
#include "sgl_kv8.h"

namespace sgl {
namespace {

struct NormArgs {
  const void *x, *res, *gate, *before, *after;
  int64_t xs, rs, gs, hs;  // elements between rows
  void *h, *y;
  void* scales;
  int64_t T;
  int H, units;  // units of 8 elements in a row, the last one may be short
  float alpha, eps, inv_h;
  int gate_type;  // -1: none
  int before_type, after_type;
  bool gate_rows;  // a gate for each element, not for each channel
  int group, mode;
  bool e8m0;
};

// 8 elements from `at` on as they lie; `n` of them are there (the others zero).  Rows may begin
// at any element, so the loads ask for no alignment beyond it (gfx950 takes them whole).
template <int DT>
struct Raw {
  uint32_t w[DT == SGL_F32 ? 8 : 4];
};
template <int DT>
__device__ __forceinline__ Raw<DT> fetch(const void* base, int64_t at, int n) {
  typedef std::conditional_t<DT == SGL_F32, uint32_t, uint16_t> E;
  const E* p = (const E*)base + at;
  Raw<DT> r;
  if (__builtin_expect(n == 8, 1)) {
    __builtin_memcpy(r.w, p, sizeof(r.w));
  } else {
    E e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < n ? p[i] : (E)0;
    __builtin_memcpy(r.w, e, sizeof(r.w));
  }
  return r;
}
template <int DT>
__device__ __forceinline__ void widen(const Raw<DT>& r, float* f) {
  uint4 raw[DT == SGL_F32 ? 2 : 1];
  __builtin_memcpy(raw, r.w, sizeof(r.w));
  widen8<DT>(raw, f);
}
__device__ __forceinline__ void fetch_any(int type, const void* base, int64_t at, int n, float* f) {
  if (type == SGL_F32)
    widen<SGL_F32>(fetch<SGL_F32>(base, at, n), f);
  else if (type == SGL_BF16)
    widen<SGL_BF16>(fetch<SGL_BF16>(base, at, n), f);
  else
    widen<SGL_F16>(fetch<SGL_F16>(base, at, n), f);
}
template <int DT>
__device__ __forceinline__ void put(void* base, int64_t at, int n, const float* f) {
  typedef std::conditional_t<DT == SGL_F32, uint32_t, uint16_t> E;
  E* p = (E*)base + at;
  Raw<DT> r;
  if constexpr (DT == SGL_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = f32_bits(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = pack2<DT>(f[2 * i], f[2 * i + 1]);
  }
  if (__builtin_expect(n == 8, 1)) {
    __builtin_memcpy(p, r.w, sizeof(r.w));
  } else {
    E e[8];
    __builtin_memcpy(e, r.w, sizeof(r.w));
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = e[i];
  }
}

// Sum over a wavefront by DPP moves, the same in every lane.
__device__ __forceinline__ float wave_sum(float v) {
  auto move = [](float x, auto ctrl, auto rows) {
    return bits_f32((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f32_bits(x), decltype(ctrl)::value,
                                                          decltype(rows)::value, 0xF, false));
  };
  typedef std::integral_constant<int, 0xF> all;
  v += move(v, std::integral_constant<int, 0x111>{}, all{});  // row_shr 1, 2, 4, 8
  v += move(v, std::integral_constant<int, 0x112>{}, all{});
  v += move(v, std::integral_constant<int, 0x114>{}, all{});
  v += move(v, std::integral_constant<int, 0x118>{}, all{});
  v += move(v, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});  // row_bcast 15
  v += move(v, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});  // row_bcast 31
  return bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(v), 63));
}

// DT: type of x and y; RT: of the residual stream; IT: units of a thread.  KEEP: the weights and
// the next row in registers, which 1024 threads (rows above 8192 elements) leave no room for.
template <int DT, int RT, int IT, bool KEEP, bool QUANT>
__global__ __launch_bounds__(KEEP ? 256 * IT : 1024) void norm_kernel(const NormArgs a) {
  __shared__ float part[4][16];
  const int waves = (int)(blockDim.x >> 6), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int at[IT], n[IT];
  float before[KEEP ? IT : 1][8], after[KEEP ? IT : 1][8], gate[KEEP ? IT : 1][8];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int u = k * (int)blockDim.x + (int)threadIdx.x;
    at[k] = 8 * u;
    const int left = a.H - 8 * u;
    n[k] = u >= a.units ? 0 : left < 8 ? left : 8;
    if (!KEEP || n[k] == 0) continue;
    if (a.before) fetch_any(a.before_type, a.before, at[k], n[k], before[KEEP ? k : 0]);
    if (a.after) fetch_any(a.after_type, a.after, at[k], n[k], after[KEEP ? k : 0]);
    if (a.gate_type >= 0 && !a.gate_rows) fetch_any(a.gate_type, a.gate, at[k], n[k], gate[KEEP ? k : 0]);
  }
  auto sum_over_row = [&](float v, int slot) {
    v = wave_sum(v);
    if (waves == 1) return v;
    if ((threadIdx.x & 63) == 0) part[slot][wave] = v;
    __syncthreads();  // (four slots in turn: nobody writes one that another still reads)
    float s = 0.0f;
    for (int i = 0; i < waves; ++i) s += part[slot][i];
    return s;
  };
  Raw<DT> x[IT];
  Raw<RT> r[IT];
  auto load = [&](int64_t t) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      if (n[k] == 0) continue;
      x[k] = fetch<DT>(a.x, t * a.xs + at[k], n[k]);
      r[k] = fetch<RT>(a.res, t * a.rs + at[k], n[k]);
    }
  };
  int slot = 0;
  if (KEEP && (int64_t)blockIdx.x < a.T) load(blockIdx.x);
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    float u[IT][8], h[IT][8];
    if (!KEEP) load(t);
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      if (n[k] == 0) continue;
      widen<DT>(x[k], u[k]);
      widen<RT>(r[k], h[k]);
      if (KEEP && a.gate_rows) fetch_any(a.gate_type, a.gate, t * a.gs + at[k], n[k], gate[k]);
    }
    if (KEEP && t + gridDim.x < a.T) load(t + gridDim.x);
    if (a.after) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < IT; ++k)
        if (n[k])
#pragma unroll
          for (int i = 0; i < 8; ++i) s = __builtin_fmaf(u[k][i], u[k][i], s);
      const float f = 1.0f / __builtin_sqrtf(__builtin_fmaf(sum_over_row(s, slot), a.inv_h, a.eps));
      slot = (slot + 1) & 3;
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        if (n[k] == 0) continue;
        float* w = after[KEEP ? k : 0];
        if (!KEEP) fetch_any(a.after_type, a.after, at[k], n[k], w);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[k][i] = u[k][i] * f * w[i];
      }
    }
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      if (n[k] == 0) continue;
      float* w = gate[KEEP ? k : 0];
      if (!KEEP && a.gate_type >= 0) fetch_any(a.gate_type, a.gate, (a.gate_rows ? t * a.gs : 0) + at[k], n[k], w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (a.gate_type >= 0) u[k][i] *= w[i];
        h[k][i] = __builtin_fmaf(a.alpha, u[k][i], h[k][i]);
      }
      put<RT>(a.h, t * a.hs + at[k], n[k], h[k]);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n[k]) s = __builtin_fmaf(h[k][i], h[k][i], s);
    }
    if (!a.before) continue;
    const float f = 1.0f / __builtin_sqrtf(__builtin_fmaf(sum_over_row(s, slot), a.inv_h, a.eps));
    slot = (slot + 1) & 3;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      if (n[k] == 0) continue;
      float y[8];
      float* w = before[KEEP ? k : 0];
      if (!KEEP) fetch_any(a.before_type, a.before, at[k], n[k], w);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = h[k][i] * f * w[i];
      if constexpr (!QUANT) {
        put<DT>(a.y, t * a.H + at[k], n[k], y);
      } else {
        // a group is 4, 8 or 16 neighbouring lanes, all of them on the row or none
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = __builtin_elementwise_maximum(most, __builtin_fabsf(y[i]));
        most = a.group == 128 ? lane_group_max<16>(most) : a.group == 64 ? lane_group_max<8>(most) : lane_group_max<4>(most);
        float sf;
        uint2 q;
        auto code = [&](auto mode) __attribute__((always_inline)) {
          sf = group_scale(decltype(mode)::value, most);
          q = quant8_e4m3(decltype(mode)::value, y, sf);
        };
        if (a.mode == SCALE_TORCH_FP32)
          code(std::integral_constant<int, SCALE_TORCH_FP32>{});
        else if (a.mode == SCALE_TORCH_UE8M0)
          code(std::integral_constant<int, SCALE_TORCH_UE8M0>{});
        else if (a.mode == SCALE_TILELANG_FP32)
          code(std::integral_constant<int, SCALE_TILELANG_FP32>{});
        else
          code(std::integral_constant<int, SCALE_TILELANG_UE8M0>{});
        *reinterpret_cast<uint2*>((uint8_t*)a.y + t * a.H + at[k]) = q;
        if (at[k] % a.group == 0) {
          const int64_t g = t * (a.H / a.group) + at[k] / a.group;
          if (a.e8m0)
            ((uint8_t*)a.scales)[g] = pow2_to_e8m0(sf);
          else
            ((float*)a.scales)[g] = sf;
        }
      }
    }
  }
}

template <int DT, int RT, int IT, bool KEEP>
void launch_norm(const NormArgs& a, const NormPlan& p, bool quant, hipStream_t st) {
  if (quant)
    norm_kernel<DT, RT, IT, KEEP, true><<<(unsigned)p.grid, (unsigned)p.threads, 0, st>>>(a);
  else
    norm_kernel<DT, RT, IT, KEEP, false><<<(unsigned)p.grid, (unsigned)p.threads, 0, st>>>(a);
}

template <int DT, int RT>
void launch_norm_as(const NormArgs& a, bool quant, hipStream_t st) {
  const NormPlan p = norm_plan(a.T, a.units, device_cu_count());
  if (p.units == 1)
    launch_norm<DT, RT, 1, true>(a, p, quant, st);
  else if (p.threads <= 512)
    launch_norm<DT, RT, 2, true>(a, p, quant, st);
  else
    launch_norm<DT, RT, 2, false>(a, p, quant, st);
}

}  // namespace
}  // namespace sgl

extern "C" {

int sgl_residual_norm(const void* x, int dtype, int64_t T, int64_t H, int64_t x_stride, const void* residual,
                      int residual_dtype, int64_t residual_stride, const void* after, int after_dtype,
                      const void* gate, int gate_dtype, int gate_rows, int64_t gate_stride, float scale,
                      const void* before, int before_dtype, float eps, void* h, int64_t h_stride, void* y, int quant,
                      void* scales, int group, int scale_mode, int scale_e8m0, sgl_stream_t stream) {
  auto is_float = [](int t) { return t == SGL_BF16 || t == SGL_F16 || t == SGL_F32; };
  SGL_REQUIRE(is_float(dtype) && (residual_dtype == dtype || residual_dtype == SGL_F32),
              "residual_norm: dtype %d with a residual of %d", dtype, residual_dtype);
  SGL_REQUIRE((!after || is_float(after_dtype)) && (!before || is_float(before_dtype)) &&
                  (!gate || is_float(gate_dtype)),
              "residual_norm: dtype of a weight or gate");
  SGL_REQUIRE(T >= 0 && T < (1ll << 40) && H >= 1 && H <= sgl::kNormMost,
              "residual_norm: T=%lld H=%lld out of range (H at most %lld)", (long long)T, (long long)H,
              (long long)sgl::kNormMost);
  SGL_REQUIRE(eps >= 0.0f && eps < __builtin_huge_valf(), "residual_norm: eps must be finite and not negative");
  if (quant) {
    SGL_REQUIRE(before, "residual_norm: codes are of the norm before the next block, which is missing");
    SGL_REQUIRE(group == 32 || group == 64 || group == 128, "residual_norm: group=%d must be 32, 64 or 128", group);
    SGL_REQUIRE(H % group == 0, "residual_norm: H=%lld must be divisible by the group (%d)", (long long)H, group);
    SGL_REQUIRE(scale_mode >= SGL_SCALE_TORCH_FP32 && scale_mode <= SGL_SCALE_TILELANG_UE8M0,
                "residual_norm: scale_mode %d", scale_mode);
    SGL_REQUIRE(!scale_e8m0 || scale_mode == SGL_SCALE_TORCH_UE8M0 || scale_mode == SGL_SCALE_TILELANG_UE8M0,
                "residual_norm: e8m0 scales need a power-of-two scale mode");
  }
  if (T == 0) return SGL_OK;
  SGL_REQUIRE(x && residual && h && (y || !before) && (scales || !quant), "residual_norm: null pointer");
  auto fits = [](const void* p, int t) { return sgl::aligned(p, t == SGL_F32 ? 4 : 2); };
  SGL_REQUIRE(fits(x, dtype) && fits(residual, residual_dtype) && fits(h, residual_dtype) &&
                  (!after || fits(after, after_dtype)) && (!before || fits(before, before_dtype)) &&
                  (!gate || fits(gate, gate_dtype)),
              "residual_norm: misaligned pointer");
  SGL_REQUIRE(!before || (quant ? sgl::aligned(y, 8) && sgl::aligned(scales, scale_e8m0 ? 1 : 4) : fits(y, dtype)),
              "residual_norm: misaligned output");
  sgl::NormArgs a;
  a.x = x;
  a.res = residual;
  a.gate = gate;
  a.before = before;
  a.after = after;
  a.xs = x_stride;
  a.rs = residual_stride;
  a.gs = gate_stride;
  a.hs = h_stride;
  a.h = h;
  a.y = y;
  a.scales = scales;
  a.T = T;
  a.H = (int)H;
  a.units = (int)sgl::ceil_div(H, 8);
  a.alpha = scale;
  a.eps = eps;
  a.inv_h = 1.0f / (float)H;
  a.gate_type = gate ? gate_dtype : -1;
  a.before_type = before_dtype;
  a.after_type = after_dtype;
  a.gate_rows = gate && gate_rows;
  a.group = group;
  a.mode = scale_mode;
  a.e8m0 = scale_e8m0 != 0;
  const hipStream_t st = (hipStream_t)stream;
  const bool q = quant != 0;
  if (dtype == SGL_F32)
    sgl::launch_norm_as<SGL_F32, SGL_F32>(a, q, st);
  else if (dtype == SGL_BF16 && residual_dtype == SGL_F32)
    sgl::launch_norm_as<SGL_BF16, SGL_F32>(a, q, st);
  else if (dtype == SGL_BF16)
    sgl::launch_norm_as<SGL_BF16, SGL_BF16>(a, q, st);
  else if (residual_dtype == SGL_F32)
    sgl::launch_norm_as<SGL_F16, SGL_F32>(a, q, st);
  else
    sgl::launch_norm_as<SGL_F16, SGL_F16>(a, q, st);
  return sgl::check_launch("residual_norm");
}

}  // extern "C"
