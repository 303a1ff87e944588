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
// the sums; the weights and a gate of channels stay in registers.  bf16, both norms: 16384 rows of
// 4096 with codes 78 to 81 us on three sets of inputs in turn, 5.8 to 6.0 TB/s of what it reads and writes, 82 to
// 94 us on inputs just written; 1900 of 7168 with an fp32 residual and a gate of each element 35 and 40 us, 5.4
// and 4.8 TB/s; 8 rows with one norm 3.9 us, two sums over a workgroup behind one another and the way to memory.
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

// 8 elements from `at` on as they lie; `n` of them are there (the others zero; without TAIL all are).  Rows may begin
// at any element, so the loads ask for no alignment beyond it (gfx950 takes them whole).
template <int DT>
struct Raw {
  uint32_t w[DT == SGL_F32 ? 8 : 4];
};
// ONCE: with the nontemporal policy, for lines that one load takes whole (16-bit elements).
template <int DT, bool TAIL, bool ONCE = false>
__device__ __forceinline__ Raw<DT> fetch(const void* base, int64_t at, int n) {
  typedef std::conditional_t<DT == SGL_F32, uint32_t, uint16_t> E;
  const E* p = (const E*)base + at;
  Raw<DT> r;
  if (!TAIL || __builtin_expect(n == 8, 1)) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    typedef u4 u4h __attribute__((aligned(2)));
    typedef u4 u4w __attribute__((aligned(4)));
    typedef std::conditional_t<DT == SGL_F32, u4w, u4h> u4v;
#pragma unroll
    for (int i = 0; i < (int)sizeof(r.w) / 16; ++i) {
      const u4 v = ONCE ? __builtin_nontemporal_load((const u4v*)p + i) : ((const u4v*)p)[i];
      __builtin_memcpy(r.w + 4 * i, &v, 16);
    }
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
template <bool TAIL>
__device__ __forceinline__ void fetch_any(int type, const void* base, int64_t at, int n, float* f) {
  if (type == SGL_F32)
    widen<SGL_F32>(fetch<SGL_F32, TAIL>(base, at, n), f);
  else if (type == SGL_BF16)
    widen<SGL_BF16>(fetch<SGL_BF16, TAIL>(base, at, n), f);
  else
    widen<SGL_F16>(fetch<SGL_F16, TAIL>(base, at, n), f);
}
template <int DT, bool TAIL>
__device__ __forceinline__ void put(void* base, int64_t at, int n, const float* f) {
  typedef std::conditional_t<DT == SGL_F32, uint32_t, uint16_t> E;
  E* p = (E*)base + at;
  Raw<DT> r;
  if constexpr (DT == SGL_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = f32_bits(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = DT == SGL_BF16 ? pk2_bf16(f[2 * i], f[2 * i + 1]) : pack2<DT>(f[2 * i], f[2 * i + 1]);
  }
  if (!TAIL || __builtin_expect(n == 8, 1)) {
    __builtin_memcpy(p, r.w, sizeof(r.w));
  } else {
    E e[8];
    __builtin_memcpy(e, r.w, sizeof(r.w));
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = e[i];
  }
}

// Sums by DPP moves: of 16 lanes in the last of them, then of a wavefront, the same in every lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved(float x) {
  return bits_f32((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f32_bits(x), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ float lane_of(float v, int lane) {
  return bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(v), lane));
}
__device__ __forceinline__ float row_sum(float v) {
  v += moved<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
  v = row_sum(v);
  v += moved<0x142, 0xA>(v);  // row_bcast 15
  v += moved<0x143, 0xC>(v);  // row_bcast 31
  return lane_of(v, 63);
}

// DT: type of x and y; RT: of the residual stream; IT: units of a thread.  KEEP: the weights in
// registers and the next row's loads in flight, which two units leave no room for.  ONCE: the rows do
// not fit the last-level cache, and pass it by.  TAIL: H is no multiple of 8.  Without it no load
// stands under a branch, or the waits for one would be waits for the next row's loads too:
// threads behind the row's end load its first unit, and a last row again.
template <int DT, int RT, int IT, bool ONCE, bool TAIL, bool QUANT>
__global__ __launch_bounds__(1024) void norm_kernel(const NormArgs a) {
  constexpr bool KEEP = IT == 1;
  __shared__ float part[4][16];
  const int waves = (int)(blockDim.x >> 6), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int at[IT], n[IT];
  float before[KEEP ? IT : 1][8], factor[KEEP ? IT : 1][8];  // factor: after * gate, a row's gate apart
  // What u is multiplied by, but for a gate of each element.
  auto load_factor = [&](int k, float* w) __attribute__((always_inline)) {
    if (a.after) fetch_any<TAIL>(a.after_type, a.after, at[k], n[k], w);
    if (a.gate_type >= 0 && !a.gate_rows) {
      float g[8];
      fetch_any<TAIL>(a.gate_type, a.gate, at[k], n[k], g);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = a.after ? w[i] * g[i] : g[i];
    }
  };
  const bool scaled = a.after || (a.gate_type >= 0 && !a.gate_rows);
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int u = k * (int)blockDim.x + (int)threadIdx.x;
    const int left = a.H - 8 * u;
    n[k] = u >= a.units ? 0 : left < 8 ? left : 8;
    at[k] = n[k] ? 8 * u : 0;
    if (!KEEP) continue;
    if (a.before) fetch_any<TAIL>(a.before_type, a.before, at[k], n[k], before[k]);
    load_factor(k, factor[k]);
  }
  int slot = 0;
  auto sum_over_row = [&](float v) {
    v = wave_sum(v);
    if (waves == 1) return v;
    if ((threadIdx.x & 63) == 0) part[slot][wave] = v;
    // (no wait for memory; four slots in turn: nobody writes one that another still reads)
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int i = (int)(threadIdx.x & 15);
    const float s = part[slot][i];
    slot = (slot + 1) & 3;
    return lane_of(row_sum(i < waves ? s : 0.0f), 15);
  };
  Raw<DT> x[IT];
  Raw<RT> r[IT];
  auto load = [&](int64_t t) __attribute__((always_inline)) {
    t = t < a.T ? t : a.T - 1;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      x[k] = fetch<DT, TAIL, ONCE>(a.x, t * a.xs + at[k], n[k]);
      r[k] = fetch<RT, TAIL, ONCE>(a.res, t * a.rs + at[k], n[k]);
    }
  };
  if (KEEP) load(blockIdx.x);
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    float u[IT][8], h[IT][8];
    if (!KEEP) load(t);
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      widen<DT>(x[k], u[k]);
      widen<RT>(r[k], h[k]);
    }
    if (KEEP) load(t + gridDim.x);
    float f = a.alpha;
    if (a.after) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        float q = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) q = __builtin_fmaf(u[k][i], u[k][i], q);
        s += n[k] ? q : 0.0f;
      }
      f *= 1.0f / __builtin_sqrtf(__builtin_fmaf(sum_over_row(s), a.inv_h, a.eps));
    }
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      if (a.gate_rows) {
        float g[8];
        fetch_any<TAIL>(a.gate_type, a.gate, t * a.gs + at[k], n[k], g);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[k][i] *= g[i];
      }
      if (scaled) {
        float* w = factor[KEEP ? k : 0];
        if (!KEEP) load_factor(k, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[k][i] *= w[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) h[k][i] = __builtin_fmaf(f, u[k][i], h[k][i]);
      if (n[k]) put<RT, TAIL>(a.h, t * a.hs + at[k], n[k], h[k]);
      float q = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) q = !TAIL || i < n[k] ? __builtin_fmaf(h[k][i], h[k][i], q) : q;
      s += n[k] ? q : 0.0f;
    }
    if (!a.before) continue;
    f = 1.0f / __builtin_sqrtf(__builtin_fmaf(sum_over_row(s), a.inv_h, a.eps));
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      float* w = before[KEEP ? k : 0];
      if (!KEEP) fetch_any<TAIL>(a.before_type, a.before, at[k], n[k], w);
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = h[k][i] * f * w[i];
      if constexpr (!QUANT) {
        if (n[k]) put<DT, TAIL>(a.y, t * a.H + at[k], n[k], y);
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
          float v[8];
          quant_scale<8>(decltype(mode)::value, y, sf, v);
          if (__builtin_expect(most < __builtin_huge_valf(), 1))  // (a NaN's sign is the conversion's own)
            q = make_uint2(pk4_e4m3(v[0], v[1], v[2], v[3]), pk4_e4m3(v[4], v[5], v[6], v[7]));
          else
            q = make_uint2(pk4_e4m3_exact(v[0], v[1], v[2], v[3]), pk4_e4m3_exact(v[4], v[5], v[6], v[7]));
        };
        if (a.mode == SCALE_TORCH_FP32)
          code(std::integral_constant<int, SCALE_TORCH_FP32>{});
        else if (a.mode == SCALE_TORCH_UE8M0)
          code(std::integral_constant<int, SCALE_TORCH_UE8M0>{});
        else if (a.mode == SCALE_TILELANG_FP32)
          code(std::integral_constant<int, SCALE_TILELANG_FP32>{});
        else
          code(std::integral_constant<int, SCALE_TILELANG_UE8M0>{});
        if (n[k]) {
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
}

template <int DT, int RT, int IT, bool ONCE>
void launch_norm(const NormArgs& a, const NormPlan& p, bool quant, hipStream_t st) {
  const dim3 grid((unsigned)p.grid), threads((unsigned)p.threads);
  if (quant)  // (groups of 32 at least: no tail)
    norm_kernel<DT, RT, IT, ONCE, false, true><<<grid, threads, 0, st>>>(a);
  else if (a.H % 8 == 0)
    norm_kernel<DT, RT, IT, ONCE, false, false><<<grid, threads, 0, st>>>(a);
  else
    norm_kernel<DT, RT, IT, ONCE, true, false><<<grid, threads, 0, st>>>(a);
}

template <int DT, int RT>
void launch_norm_as(const NormArgs& a, bool quant, hipStream_t st) {
  const NormPlan p = norm_plan(a.T, a.units, device_cu_count());
  if (p.units == 1) {
    if constexpr (RT != SGL_F32) {
      if (norm_once(a.T, a.H)) {
        launch_norm<DT, RT, 1, true>(a, p, quant, st);
        return;
      }
    }
    launch_norm<DT, RT, 1, false>(a, p, quant, st);
  } else {
    launch_norm<DT, RT, 2, false>(a, p, quant, st);
  }
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
