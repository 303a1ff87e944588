// Rotary positions: pairs (a, b) of a head's elements turned by the angle
// p f_i of the row's position p,
//   a' = a c - b s,  b' = b c + a s,  (c, s) = m (cos p f_i, sin p f_i),
// pair i being (i, i + rot / 2) (halves) or (2 i, 2 i + 1) (interleaved) of the
// rot elements from `offset` on; the others are copied.  The inverse turns by
// -p f_i, which is also the gradient.  fp32 throughout, rounded once.
//
// Bound by HBM: an element is read and written once, the table's row once for
// all heads of a token.  A thread takes 2 x 8 elements (16-byte accesses; both
// chunks of its pairs, so that the rotation may be done in place) of several
// heads with the same cos and sin in registers.  16384 tokens of 32 heads of 128:
// 51 to 54 us, 5.2 TB/s, a large copy's rate.
#include "sgl_kv8.h"

namespace sgl {
namespace {

// angles in 64 bits: at position 10^6 a 32-bit angle would be 0.03 radians off
__global__ __launch_bounds__(256) void rotary_table_kernel(const double* freq, double length, int64_t n,
                                                           int pairs, float2* table) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n * pairs) return;
  const int64_t p = i / pairs;
  double s, c;
  sincos((double)p * freq[i - p * pairs], &s, &c);
  table[i] = make_float2((float)(c * length), (float)(s * length));
}

struct RotaryArgs {
  const void* x;
  void* out;
  int64_t xt, xh, ot, oh;  // elements between tokens, heads
  const float* table;
  int64_t n_positions;
  const void* positions;
  int T, H, D, rot, offset;
  int units;    // a head's units of 2 VEC elements that there is work on
  int hsplit;   // threads that share a unit's heads
  bool pos64, interleaved, inverse;
};

constexpr int kHeads = 4;  // heads of a thread in flight

template <int DT, int VEC>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
  const uint32_t per = (uint32_t)(a.units * a.hsplit);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = i / per;
  if (t >= a.T) return;
  const uint32_t j = (uint32_t)(i - t * per);
  const int hs = (int)(j / (uint32_t)a.units), u = (int)(j - (uint32_t)hs * a.units);
  const int rot_units = a.rot / (2 * VEC);
  int e0, e1;  // the unit's two chunks of VEC elements
  bool two = true;
  if (u < rot_units) {
    e0 = a.offset + (a.interleaved ? 2 * VEC : VEC) * u;
    e1 = e0 + (a.interleaved ? VEC : a.rot / 2);
  } else {
    const int c = 2 * VEC * (u - rot_units), rest = a.D - a.rot;
    e0 = c < a.offset ? c : c + a.rot;
    e1 = c + VEC < a.offset ? c + VEC : c + VEC + a.rot;
    two = c + VEC < rest;
  }
  float cs[VEC], sn[VEC];
  bool turn = false;
  if (u < rot_units) {
    const int64_t p = a.pos64 ? ((const int64_t*)a.positions)[t] : ((const int32_t*)a.positions)[t];
    turn = p >= 0;
    if (turn) load_turn<VEC>(a.table, a.n_positions, a.rot / 2, p, VEC * u, a.inverse, cs, sn);
  }
  auto load = [&](int64_t at, float* f) {
    if constexpr (VEC == 8) {
      load8<DT>(a.x, at, f);
    } else if constexpr (DT == SGL_F32) {
      f[0] = ((const float*)a.x)[at];
    } else {
      const uint16_t w = ((const uint16_t*)a.x)[at];
      f[0] = DT == SGL_BF16 ? bf16_to_f32(w) : (float)__builtin_bit_cast(_Float16, w);
    }
  };
  auto store = [&](int64_t at, const float* f) {
    if constexpr (VEC == 8) {
      store8<DT>(a.out, at, f);
    } else if constexpr (DT == SGL_F32) {
      ((float*)a.out)[at] = f[0];
    } else {
      ((uint16_t*)a.out)[at] = (uint16_t)pack2<DT>(f[0], 0.0f);
    }
  };
  for (int h0 = hs; h0 < a.H; h0 += kHeads * a.hsplit) {
    float x[kHeads][2][VEC];
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
      const int h = h0 + k * a.hsplit;
      if (h < a.H) {
        load(t * a.xt + h * a.xh + e0, x[k][0]);
        if (two) load(t * a.xt + h * a.xh + e1, x[k][1]);
      }
    }
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
      const int h = h0 + k * a.hsplit;
      if (h < a.H) {
        if (turn) {
          if (VEC == 8 && a.interleaved) {
            float p[VEC], q[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
              p[v] = x[k][v / (VEC / 2 > 0 ? VEC / 2 : 1)][2 * v % VEC];
              q[v] = x[k][v / (VEC / 2 > 0 ? VEC / 2 : 1)][(2 * v + 1) % VEC];
            }
            rotate_pairs<VEC>(p, q, cs, sn);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
              x[k][v / (VEC / 2 > 0 ? VEC / 2 : 1)][2 * v % VEC] = p[v];
              x[k][v / (VEC / 2 > 0 ? VEC / 2 : 1)][(2 * v + 1) % VEC] = q[v];
            }
          } else {
            rotate_pairs<VEC>(x[k][0], x[k][1], cs, sn);
          }
        }
        store(t * a.ot + h * a.oh + e0, x[k][0]);
        if (two) store(t * a.ot + h * a.oh + e1, x[k][1]);
      }
    }
  }
}

template <int DT>
void launch_rotary(const RotaryArgs& a, bool vec, hipStream_t st) {
  const int64_t threads = (int64_t)a.T * a.units * a.hsplit;
  const dim3 grid((unsigned)ceil_div(threads, 256));
  if (vec)
    rotary_kernel<DT, 8><<<grid, 256, 0, st>>>(a);
  else
    rotary_kernel<DT, 1><<<grid, 256, 0, st>>>(a);
}

}  // namespace
}  // namespace sgl

extern "C" {

int sgl_rotary_table(const double* freq, double length, int64_t n_positions, int rot_dim, float* table,
                     sgl_stream_t stream) {
  SGL_REQUIRE(rot_dim >= 2 && rot_dim % 2 == 0 && rot_dim <= 4096, "rotary_table: rot_dim=%d must be even, 2 to 4096",
              rot_dim);
  SGL_REQUIRE(n_positions >= 0 && n_positions <= (1ll << 31) - 1, "rotary_table: n_positions=%lld out of range",
              (long long)n_positions);
  if (n_positions == 0) return SGL_OK;
  SGL_REQUIRE(freq && table, "rotary_table: null pointer");
  SGL_REQUIRE(sgl::aligned(table, 8), "rotary_table: table must be 8-byte aligned");
  const int64_t n = n_positions * (rot_dim / 2);
  SGL_REQUIRE(n <= 256ll * 0x7FFFFFFF, "rotary_table: too large");
  sgl::rotary_table_kernel<<<(unsigned)sgl::ceil_div(n, 256), 256, 0, (hipStream_t)stream>>>(
      freq, length, n_positions, rot_dim / 2, (float2*)table);
  return sgl::check_launch("rotary_table");
}

int sgl_rotary(const void* x, int dtype, int64_t T, int H, int D, int64_t x_token_stride, int64_t x_head_stride,
               const float* table, int64_t n_positions, int rot_dim, int offset, const void* positions,
               int positions_int64, int interleaved, int inverse, void* out, int64_t out_token_stride,
               int64_t out_head_stride, sgl_stream_t stream) {
  SGL_REQUIRE(dtype == SGL_BF16 || dtype == SGL_F16 || dtype == SGL_F32, "rotary: dtype %d", dtype);
  SGL_REQUIRE(T >= 0 && T <= 0x7FFFFFFF && H >= 0 && H <= 65536 && D >= 1 && D <= 65536,
              "rotary: T=%lld H=%d D=%d out of range", (long long)T, H, D);
  SGL_REQUIRE(rot_dim >= 2 && rot_dim % 2 == 0 && offset >= 0 && offset + rot_dim <= D,
              "rotary: rot_dim=%d must be even and fit at offset %d into D=%d", rot_dim, offset, D);
  SGL_REQUIRE(n_positions >= 1, "rotary: the table has no positions");
  if (T == 0 || H == 0) return SGL_OK;
  SGL_REQUIRE(x && table && positions && out, "rotary: null pointer");
  SGL_REQUIRE(sgl::aligned(table, 8), "rotary: table must be 8-byte aligned");
  const int size = dtype == SGL_F32 ? 4 : 2;
  SGL_REQUIRE(sgl::aligned(x, size) && sgl::aligned(out, size), "rotary: misaligned pointer");
  const bool in_place = x == out;
  SGL_REQUIRE(!in_place || (x_token_stride == out_token_stride && x_head_stride == out_head_stride),
              "rotary: in place the strides of x and out must be the same");
  const bool vec = rot_dim % 16 == 0 && offset % 8 == 0 && D % 8 == 0 && sgl::aligned(x, 16) &&
                   sgl::aligned(out, 16) && sgl::aligned(table, 16) && x_token_stride * size % 16 == 0 &&
                   x_head_stride * size % 16 == 0 && out_token_stride * size % 16 == 0 &&
                   out_head_stride * size % 16 == 0;
  sgl::RotaryArgs a;
  a.x = x;
  a.out = out;
  a.xt = x_token_stride;
  a.xh = x_head_stride;
  a.ot = out_token_stride;
  a.oh = out_head_stride;
  a.table = table;
  a.n_positions = n_positions;
  a.positions = positions;
  a.T = (int)T;
  a.H = H;
  a.D = D;
  a.rot = rot_dim;
  a.offset = offset;
  a.pos64 = positions_int64 != 0;
  a.interleaved = interleaved != 0;
  a.inverse = inverse != 0;
  const int width = vec ? 16 : 2;
  a.units = rot_dim / width + (in_place ? 0 : (D - rot_dim + width - 1) / width);
  a.hsplit = sgl::rotary_head_threads(T, H, a.units, sgl::device_cu_count());
  SGL_REQUIRE((int64_t)a.T * a.units * a.hsplit <= 256ll * 0x7FFFFFFF, "rotary: too large");
  if (dtype == SGL_BF16)
    sgl::launch_rotary<SGL_BF16>(a, vec, (hipStream_t)stream);
  else if (dtype == SGL_F16)
    sgl::launch_rotary<SGL_F16>(a, vec, (hipStream_t)stream);
  else
    sgl::launch_rotary<SGL_F32>(a, vec, (hipStream_t)stream);
  return sgl::check_launch("rotary");
}

}  // extern "C"
