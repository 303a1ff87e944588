// What the kernels of the 8-bit paged cache (kv8.hip, kv8_attn.hip,
// kv8_prefill.hip) share.  Not part of the C ABI.
//
// The cache: e4m3 codes [n_pages, Hkv, page, D] for keys and values, one fp32
// scale for every `block` tokens of a page and head [n_pages, Hkv, page / block].
// Pages and blocks are powers of two of at least 16 tokens, so 16 tokens that
// start at a multiple of 16 (a granule) share page and scale.
#pragma once

#include "sgl_common.h"
#include "sgl_numeric.h"
#include "sgl_rules.h"

namespace sgl {

// The limits of a cache: heads, head dim, pages.
inline int kv8_check_cache(const char* what, int Hkv, int D, int page, int block, int64_t n_pages, int64_t row_pages) {
  SGL_REQUIRE(Hkv >= 1 && Hkv <= 4096, "%s: Hkv=%d out of range", what, Hkv);
  SGL_REQUIRE(D >= 16 && D <= 256 && D % 16 == 0, "%s: D=%d must be a multiple of 16, at most 256", what, D);
  SGL_REQUIRE(page >= 16 && page <= 1024 && (page & (page - 1)) == 0,
              "%s: page_size=%d must be a power of two, 16 to 1024", what, page);
  SGL_REQUIRE(block >= 16 && block <= 128 && block <= page && (block & (block - 1)) == 0,
              "%s: block=%d must be a power of two, 16 to 128, and at most the page (%d)", what, block, page);
  SGL_REQUIRE(n_pages >= 1 && n_pages <= 0x7FFFFFFF, "%s: n_pages=%lld out of range", what, (long long)n_pages);
  SGL_REQUIRE(row_pages >= 1 && row_pages * page <= (1 << 30), "%s: %lld pages of %d tokens a sequence: too many",
              what, (long long)row_pages, page);
  return SGL_OK;
}

// Eight elements of a row as fp32.
template <int DT>
__device__ __forceinline__ void widen8(const uint4* raw, float* f) {
  if constexpr (DT == SGL_F32) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[4 * i] = bits_f32(raw[i].x);
      f[4 * i + 1] = bits_f32(raw[i].y);
      f[4 * i + 2] = bits_f32(raw[i].z);
      f[4 * i + 3] = bits_f32(raw[i].w);
    }
  } else {
    const uint32_t v[4] = {raw->x, raw->y, raw->z, raw->w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == SGL_BF16) {
        f[2 * i] = bits_f32(v[i] << 16);
        f[2 * i + 1] = bits_f32(v[i] & 0xFFFF0000u);
      } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 h = __builtin_bit_cast(h2, v[i]);
        f[2 * i] = (float)h.x;
        f[2 * i + 1] = (float)h.y;
      }
    }
  }
}
// Eight consecutive ones as they lie: 16 or 32 bytes.
template <int DT>
__device__ __forceinline__ void load_raw8(const void* base, int64_t at, uint4* raw) {
  if constexpr (DT == SGL_F32) {
    const uint4* p = reinterpret_cast<const uint4*>((const float*)base + at);
    raw[0] = p[0];
    raw[1] = p[1];
  } else {
    *raw = *reinterpret_cast<const uint4*>((const uint16_t*)base + at);
  }
}
template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t at, float* f) {
  uint4 raw[DT == SGL_F32 ? 2 : 1];
  load_raw8<DT>(base, at, raw);
  widen8<DT>(raw, f);
}

// fp32 values rounded once to the output type: torch's casts, NaN kept.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == SGL_BF16) {
    return pk2_bf16_exact(a, b);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, h2{(_Float16)a, (_Float16)b});
  }
}
template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t at, const float* f) {
  if constexpr (DT == SGL_F32) {
    float4* p = reinterpret_cast<float4*>((float*)base + at);
    p[0] = make_float4(f[0], f[1], f[2], f[3]);
    p[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *reinterpret_cast<uint4*>((uint16_t*)base + at) =
        make_uint4(pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]), pack2<DT>(f[4], f[5]), pack2<DT>(f[6], f[7]));
  }
}

// N pairs (a, b) rotated by cs[i] = (cos, sin): two products and a sum or
// difference, each rounded, so that every path gives the same bits.
template <int N>
__device__ __forceinline__ void rotate_pairs(float* a, float* b, const float* cos, const float* sin) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float x = a[i], y = b[i];
    a[i] = x * cos[i] - y * sin[i];
    b[i] = y * cos[i] + x * sin[i];
  }
}

// cos and sin of N pairs of position p >= 0.  Behind the table's last position there
// is no rotation to give: NaN.  (A negative one marks a padding row, which is not
// turned at all: by 1 and 0 an infinity would make NaN of its partner.)
template <int N>
__device__ __forceinline__ void load_turn(const float* table, int64_t n_positions, int pairs, int64_t p,
                                          int pair, bool inverse, float* cos, float* sin) {
  const bool in = p < n_positions;
  const float2* row = reinterpret_cast<const float2*>(table) + (in ? p : 0) * pairs + pair;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float2 t = row[i];
    cos[i] = t.x;
    sin[i] = inverse ? -t.y : t.y;
  }
  if (__builtin_expect(!in, 0)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      cos[i] = __builtin_nanf("");
      sin[i] = __builtin_nanf("");
    }
  }
}

// A token's positions on up to four axes, each pair turning by one of them.  All are loaded beside
// the pairs' axes and chosen in registers, so that the chain to the table is no longer than with
// one position; and without branches, so that no load waits for another (an axis too many loads
// the first again).  Behind the table, and for an axis that there is none of: NaN, as above.
// `turn` is false where any of them is negative.
constexpr int kMaxAxes = 4;
struct AxisPositions {
  int p[kMaxAxes];  // at most n_positions, which is behind the table
  bool turn;
  __device__ __forceinline__ int of(int axis, int n_positions) const {
    return axis == 0 ? p[0] : axis == 1 ? p[1] : axis == 2 ? p[2] : axis == 3 ? p[3] : n_positions;
  }
};
template <bool POS64>
__device__ __forceinline__ int64_t load_position(const void* positions, int64_t at) {
  return POS64 ? ((const int64_t*)positions)[at] : ((const int32_t*)positions)[at];
}
template <bool POS64>
__device__ __forceinline__ AxisPositions load_axis_positions(const void* positions, int n_axes, int64_t T, int64_t t,
                                                             int n_positions) {
  AxisPositions o;
  int64_t p[kMaxAxes];
#pragma unroll
  for (int a = 0; a < kMaxAxes; ++a) p[a] = load_position<POS64>(positions, (a < n_axes ? a : 0) * T + t);
  o.turn = true;
#pragma unroll
  for (int a = 0; a < kMaxAxes; ++a) {
    o.turn = o.turn & (p[a] >= 0);
    o.p[a] = a < n_axes && p[a] < n_positions ? (int)p[a] : n_positions;
  }
  return o;
}
// Sum over the lanes up to and with this one, by DPP moves: within rows of 16,
// then each row's last lane to the row behind it, then lane 31 to the upper half.
__device__ __forceinline__ int wave_incl_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast 15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast 31
  return v;
}

// A sequence's rows of the token-major inputs: [first, first + n), inside [0, T).
struct SeqRows {
  int first, n;
};
__device__ __forceinline__ SeqRows seq_rows(const int32_t* cu, int b, int T) {
  if (!cu) return {b, b < T ? 1 : 0};
  int r0 = cu[b], r1 = cu[b + 1];
  r0 = r0 < 0 ? 0 : r0 > T ? T : r0;
  r1 = r1 < r0 ? r0 : r1 > T ? T : r1;
  return {r0, r1 - r0};
}

}  // namespace sgl
