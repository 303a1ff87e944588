// New keys and values into the 8-bit paged cache, the keys rotated on the way.
//
// Tokens [start, start + n) of a sequence fall into blocks of `block` tokens of
// a page; a block and head has one power-of-two scale for its keys and one for
// its values.  Of the new values x of a block, s = kv8_scale(max |x|) over the
// finite ones, and not below the scale that the block had if it holds earlier
// tokens of the sequence; code = e4m3(x / s), NaN for a NaN or an infinity.
// Earlier tokens are written again, e4m3(code s_old / s), only where the scale
// grew: a power of two, so nothing but codes near the smallest are rounded.  Of an
// old scale that is negative or not finite they are NaN.
//
// Bound by HBM (6 bytes for an element of k and of v: 2 x 2 read, 2 x 1
// written), and beside it by the conversion (16384 tokens of 8 heads of 128: 28 us at
// 3.8 TB/s); for single tokens by the chain table entry -> old scale -> codes.
// One workgroup takes one block, head and side (keys or values), so that the
// scale is one reduction in registers and LDS and no block has two writers.
#include "sgl_kv8.h"

namespace sgl {
namespace {

struct AppendArgs {
  const void *k, *v;
  int64_t kt, kh, vt, vh;  // elements between tokens, heads
  uint8_t *kc, *vc;
  float *ks, *vs;
  const int32_t* pages;  // [B, row_pages]
  const int32_t* start;  // [B]
  const int32_t* cu;     // [B + 1] or null: one token each
  const float* table;    // or null: no rotation
  const int32_t* positions;  // [T], or of several axes [n_axes][T]; null: a token's place
  int64_t n_positions;
  int64_t n_pages;
  int T, B, Hkv, D, row_pages, page_shift, block_shift;
  int per_magic;  // i / (D / 16) = i per_magic >> 16 for i < 4096
  int rot, offset;
  bool interleaved;
  // (behind the others, so that those are loaded as they were without)
  int n_axes;
  const uint8_t* axes;  // the axis of each pair
};

// A unit of work: the new tokens of one block of one sequence.
struct Unit {
  int row0, n;  // their rows
  int at;       // position of the first
  int page;
};

// Unit u of the batch, sequences in order; n = 0 behind the last, and where a
// table does not reach or names no page of the cache.
__device__ __forceinline__ Unit find_unit(const AppendArgs& a, int u) {
  const Unit none = {0, 0, 0, 0};
  const int bs = a.block_shift;
  int b = u, before = u;
  if (a.cu) {
    const int lane = threadIdx.x & 63;
    before = 0;
    for (int b0 = 0;; b0 += 64) {
      if (b0 >= a.B) return none;
      int c = 0;
      if (b0 + lane < a.B) {
        const SeqRows r = seq_rows(a.cu, b0 + lane, a.T);
        const int st = a.start[b0 + lane];
        if (r.n > 0 && st >= 0) c = (int)((((int64_t)st + r.n - 1) >> bs) - (st >> bs)) + 1;
      }
      const int incl = wave_incl_scan(c);
      const int total = __builtin_amdgcn_readlane(incl, 63);
      if (u < before + total) {
        const int l = __builtin_ctzll(__ballot(before + incl > u));
        b = b0 + l;
        before += __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(c, l);
        break;
      }
      before += total;
    }
  }
  if (b >= a.B) return none;
  const SeqRows r = seq_rows(a.cu, b, a.T);
  const int64_t st = a.start[b];
  if (r.n <= 0 || st < 0) return none;
  const int64_t j = (st >> bs) + (u - before);  // block of the sequence
  const int64_t lo = (j << bs) > st ? (j << bs) : st;
  const int64_t hi = ((j + 1) << bs) < st + r.n ? ((j + 1) << bs) : st + r.n;
  if (hi > ((int64_t)a.row_pages << a.page_shift)) return none;
  const int page = a.pages[(int64_t)b * a.row_pages + (lo >> a.page_shift)];
  if (page < 0 || page >= a.n_pages) return none;
  return {r.first + (int)(lo - st), (int)(hi - lo), (int)lo, page};
}

// 4 values by 1 / s, a power of two, to codes (v_cvt_scalef32_pk_fp8: scaled and
// rounded in one); finite ones alone, at most 448 s.
typedef short s2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float s) {
  s2v o = {0, 0};
  o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, a, b, s, false);
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, c, d, s, true));
}
// the same of packed 16-bit values
template <int DT>
__device__ __forceinline__ uint32_t codes4(uint32_t ab, uint32_t cd, float s) {
  s2v o = {0, 0};
  if constexpr (DT == SGL_BF16) {
    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, __builtin_bit_cast(sgl_bf2, ab), s, false);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, __builtin_bit_cast(sgl_bf2, cd), s, true);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, __builtin_bit_cast(h2, ab), s, false);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, __builtin_bit_cast(h2, cd), s, true);
  }
  return __builtin_bit_cast(uint32_t, o);
}

// cos and sin of a thread's 8 pairs from `pair` on, of several axes.  Where one axis holds
// all 8 they lie side by side.  Where it does not, they are up to 8 pieces of 8 bytes in as many
// rows, and the wavefront takes them in the order of the pairs instead: the threads leave their
// entries' places in LDS, load what stands at 64 neighbouring ones at a time and leave that there.
// (8000 tokens of 8 heads of 128, the axes in turn: 25 us by themselves.)
template <int NT>
__device__ __forceinline__ void turns_of(const AppendArgs& a, const AxisPositions& at, const uint8_t* axis, int pair,
                                         float* cos, float* sin) {
  __shared__ __align__(16) float2 sTurn[NT / 64][512];
  const int lane = threadIdx.x & 63, n = (int)a.n_positions, pairs = a.rot >> 1;
  bool same = true;
#pragma unroll
  for (int i = 1; i < 8; ++i) same = same & (axis[i] == axis[0]);
  if (__ballot(at.turn && !same) == 0) {
    if (at.turn) load_turn<8>(a.table, n, pairs, at.of(axis[0], n), pair, false, cos, sin);
    return;
  }
  float2* turns = sTurn[threadIdx.x >> 6];
  int* entries = reinterpret_cast<int*>(turns);
  auto fence = [] {  // (a wavefront's LDS accesses go in order: nothing to wait for but the compiler)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  int e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int p = at.of(axis[i], n);
    e[i] = at.turn && p < n ? p * pairs + pair + i : -1;
  }
  fence();
  *reinterpret_cast<int4*>(entries + 8 * lane) = make_int4(e[0], e[1], e[2], e[3]);
  *reinterpret_cast<int4*>(entries + 8 * lane + 4) = make_int4(e[4], e[5], e[6], e[7]);
  fence();
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = entries[64 * i + lane];
  float2 w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = reinterpret_cast<const float2*>(a.table)[e[i] < 0 ? 0 : e[i]];
  fence();
#pragma unroll
  for (int i = 0; i < 8; ++i) turns[64 * i + lane] = e[i] < 0 ? make_float2(__builtin_nanf(""), __builtin_nanf("")) : w[i];
  fence();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 q = *reinterpret_cast<const float4*>(turns + 8 * lane + 2 * i);
    cos[2 * i] = q.x;
    sin[2 * i] = q.y;
    cos[2 * i + 1] = q.z;
    sin[2 * i + 1] = q.w;
  }
}

// The two chunks of 8 elements of unit u of a row: those of 8 pairs, or two of the others.
__device__ __forceinline__ void unit_chunks(const AppendArgs& a, int rot, int u, int* p0, int* p1) {
  if (u < rot >> 4) {
    *p0 = a.offset + (a.interleaved ? 16 : 8) * u;
    *p1 = *p0 + (a.interleaved ? 8 : rot >> 1);
  } else {
    const int c = 16 * (u - (rot >> 4)), off = rot ? a.offset : 0;
    *p0 = c < off ? c : c + rot;
    *p1 = c + 8 < off ? c + 8 : c + 8 + rot;
  }
}
template <int DT>
__device__ __forceinline__ void load_rows(const AppendArgs& a, const Unit& w, const void* src, int64_t st, int64_t sh,
                                          int head, int rot, int t, int u, uint4* raw) {
  int p0, p1;
  unit_chunks(a, rot, u, &p0, &p1);
  const int64_t at = (int64_t)(w.row0 + t) * st + (int64_t)head * sh;
  load_raw8<DT>(src, at + p0, raw);
  load_raw8<DT>(src, at + p1, raw + (DT == SGL_F32 ? 2 : 1));
}

// NT threads, IT units of 16 elements a thread
template <int DT, int NT, int IT, bool AXES>
__global__ __launch_bounds__(NT) void append_kernel(const AppendArgs a) {
  constexpr int RW = DT == SGL_F32 ? 2 : 1;  // 16-byte words of 8 elements
  const int head = (int)blockIdx.y >> 1;
  const bool keys = (blockIdx.y & 1) == 0;
  const Unit w = find_unit(a, (int)blockIdx.x);
  if (w.n == 0) return;
  const void* src = keys ? a.k : a.v;
  const int64_t st = keys ? a.kt : a.vt, sh = keys ? a.kh : a.vh;
  const int rot = keys ? a.rot : 0;
  const int per = a.D >> 4, rot_units = rot >> 4;
  const int count = w.n * per;
  // What is not rotated stays packed: its largest by integers, its codes in one
  // instruction for two.
  const bool packed = DT != SGL_F32 && rot == 0;

  uint32_t kept[IT][16];  // packed as they lie, or fp32
  int e0[IT], e1[IT], tok[IT];
  bool odd[IT];  // a NaN or an infinity among them
  float amax = 0.0f;
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int i = it * NT + (int)threadIdx.x;
    tok[it] = -1;
    odd[it] = false;
    const int t = i * a.per_magic >> 16, u = i - t * per;
    uint4 raw[2 * RW];
    float cs[8], sn[8];
    AxisPositions place;
    if constexpr (AXES) {
      // before the rows: loads return in order, and the table's wait for these
      const bool mine = i < count && u < rot_units;
      uint8_t axis[8];
      place.turn = false;
      if (rot_units > 0) {
        __builtin_memcpy(axis, a.axes + (mine ? 8 * u : 0), 8);
        place = load_axis_positions<false>(a.positions, a.n_axes, a.T, w.row0 + (mine ? t : 0), (int)a.n_positions);
        place.turn = place.turn && mine;
      }
      __builtin_amdgcn_sched_barrier(0);
      if (i < count) load_rows<DT>(a, w, src, st, sh, head, rot, t, u, raw);
      // (all threads of the wavefront, those without a row too)
      if (rot_units > 0) turns_of<NT>(a, place, axis, mine ? 8 * u : 0, cs, sn);
    }
    if (i < count) {
      int p0, p1;
      unit_chunks(a, rot, u, &p0, &p1);
      if constexpr (!AXES) {
        const int64_t at = (int64_t)(w.row0 + t) * st + (int64_t)head * sh;
        load_raw8<DT>(src, at + p0, raw);
        load_raw8<DT>(src, at + p1, raw + RW);
      }
      tok[it] = t;
      e0[it] = p0;
      e1[it] = p1;
      float top, x[16];
      if (packed) {
        typedef uint16_t us2 __attribute__((ext_vector_type(2)));
        us2 m = {0, 0};
#pragma unroll
        for (int v = 0; v < 2 * RW; ++v) {
          const uint32_t q[4] = {raw[v].x, raw[v].y, raw[v].z, raw[v].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) kept[it][4 * v + j] = q[j];
#pragma unroll
          for (int j = 0; j < 4; ++j) m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, q[j] & 0x7FFF7FFFu));
        }
        const uint32_t most = m.x > m.y ? m.x : m.y;
        odd[it] = most >= (DT == SGL_BF16 ? 0x7F80u : 0x7C00u);
        top = DT == SGL_BF16 ? bits_f32(most << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)most);
      } else {
        widen8<DT>(raw, x);
        widen8<DT>(raw + RW, x + 8);
        bool turn = u < rot_units;
        if constexpr (AXES) {
          turn = place.turn;
        } else {
          const int64_t pos = !turn ? -1 : a.positions ? a.positions[w.row0 + t] : w.at + t;
          turn = pos >= 0;
          if (turn) load_turn<8>(a.table, a.n_positions, a.rot >> 1, pos, 8 * u, false, cs, sn);
        }
        if (turn) {
          if (a.interleaved) {
            float p[8], q[8];
#pragma unroll
            for (int v = 0; v < 8; ++v) {
              p[v] = x[2 * v];
              q[v] = x[2 * v + 1];
            }
            rotate_pairs<8>(p, q, cs, sn);
#pragma unroll
            for (int v = 0; v < 8; ++v) {
              x[2 * v] = p[v];
              x[2 * v + 1] = q[v];
            }
          } else {
            rotate_pairs<8>(x, x + 8, cs, sn);
          }
        }
        uint32_t most = 0;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          kept[it][v] = f32_bits(x[v]);
          const uint32_t m = kept[it][v] & 0x7FFFFFFFu;
          most = m > most ? m : most;
        }
        odd[it] = most >= 0x7F800000u;
        top = bits_f32(most);
      }
      if (__builtin_expect(odd[it], 0)) {  // finite values alone
        if (packed) {
          widen8<DT>(raw, x);
          widen8<DT>(raw + RW, x + 8);
        }
        top = 0.0f;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const float m = __builtin_fabsf(x[v]);
          top = m < __builtin_huge_valf() && m > top ? m : top;
        }
      }
      amax = top > amax ? top : amax;
    }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) amax = __builtin_fmaxf(amax, __shfl_xor(amax, d, 64));

  // the block's place
  const int spot = w.at & ((1 << a.page_shift) - 1);
  const int begin = spot & ~((1 << a.block_shift) - 1);
  const int64_t line = (int64_t)w.page * a.Hkv + head;
  uint8_t* codes = (keys ? a.kc : a.vc) + (line << a.page_shift) * a.D;
  float* scale = (keys ? a.ks : a.vs) + (line << (a.page_shift - a.block_shift)) + (spot >> a.block_shift);
  const float was = spot > begin ? *scale : 0.0f;
  if constexpr (NT > 64) {
    __shared__ float part[NT / 64];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = amax;
    __syncthreads();  // (the old scale is read by then)
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) amax = __builtin_fmaxf(amax, part[i]);
  }
  float s = kv8_scale(amax);
  if (was >= s && was < __builtin_huge_valf()) {
    s = was;
  } else if (spot > begin) {
    const float inv = 1.0f / s;  // exact
    const float old = was >= 0.0f ? was : __builtin_nanf("");  // (an infinity makes NaN codes of itself)
    const int bytes = (spot - begin) * a.D;
    for (int i = 16 * (int)threadIdx.x; i < bytes; i += 16 * NT) {
      uint4* at = reinterpret_cast<uint4*>(codes + (int64_t)begin * a.D + i);
      const uint4 c = *at;
      uint32_t q[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[4];
        unpack4_e4m3(q[j], f);
        const uint32_t keep = ((((q[j] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xFFu;  // NaN codes
        const uint32_t r = pk4_e4m3(f[0] * old * inv, f[1] * old * inv, f[2] * old * inv, f[3] * old * inv);
        q[j] = (q[j] & keep) | (r & ~keep);
      }
      *at = make_uint4(q[0], q[1], q[2], q[3]);
    }
  }
  if (threadIdx.x == 0) *scale = s;
  // An old scale that this kernel did not write may be no power of two, and the packed
  // conversions take an exponent alone.
  const bool uneven = (f32_bits(s) & 0x7FFFFFu) != 0;
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    if (tok[it] >= 0) {
      uint8_t* row = codes + (int64_t)(spot + tok[it]) * a.D;
      uint32_t c[4];
      if (__builtin_expect(odd[it] || uneven, 0)) {  // an infinity becomes the NaN code, a NaN keeps its sign
        float f[16];
#pragma unroll
        for (int v = 0; v < 16; ++v) f[v] = bits_f32(kept[it][v]);
        if (packed) {
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const uint4 raw = make_uint4(kept[it][4 * v], kept[it][4 * v + 1], kept[it][4 * v + 2], kept[it][4 * v + 3]);
            widen8<DT == SGL_F32 ? SGL_BF16 : DT>(&raw, f + 8 * v);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          c[j] = pk4_e4m3_exact(f[4 * j] / s, f[4 * j + 1] / s, f[4 * j + 2] / s, f[4 * j + 3] / s);
      } else if (packed) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = codes4<DT>(kept[it][2 * j], kept[it][2 * j + 1], s);
      } else {
        const uint32_t* f = kept[it];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          c[j] = codes4(bits_f32(f[4 * j]), bits_f32(f[4 * j + 1]), bits_f32(f[4 * j + 2]), bits_f32(f[4 * j + 3]), s);
      }
      if (rot == 0) {  // the two chunks lie side by side
        *reinterpret_cast<uint4*>(row + e0[it]) = make_uint4(c[0], c[1], c[2], c[3]);
      } else {
        *reinterpret_cast<uint2*>(row + e0[it]) = make_uint2(c[0], c[1]);
        *reinterpret_cast<uint2*>(row + e1[it]) = make_uint2(c[2], c[3]);
      }
    }
  }
}

// By a unit's 16 elements: a thread each up to 512 (256 threads with two each: 31.3 us
// against 30.4 for 16384 tokens of 8 heads of 128), the small ones in small workgroups.
template <int DT, bool AXES>
void launch_append(const AppendArgs& a, int64_t units, int64_t per_unit, hipStream_t st) {
  const dim3 grid((unsigned)units, (unsigned)(2 * a.Hkv));
  if (per_unit <= 64)
    append_kernel<DT, 64, 1, AXES><<<grid, 64, 0, st>>>(a);
  else if (per_unit <= 256)
    append_kernel<DT, 256, 1, AXES><<<grid, 256, 0, st>>>(a);
  else if (per_unit <= 512)
    append_kernel<DT, 512, 1, AXES><<<grid, 512, 0, st>>>(a);
  else if (per_unit <= 1024)
    append_kernel<DT, 512, 2, AXES><<<grid, 512, 0, st>>>(a);
  else
    append_kernel<DT, 512, 4, AXES><<<grid, 512, 0, st>>>(a);
}

template <bool AXES>
int append(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
           int64_t v_head_stride, int dtype, int64_t T, int64_t B, int Hkv, int D, const int32_t* cu_tokens,
           const int32_t* start, const int32_t* block_table, int64_t row_pages, int page_size, int block,
           int64_t n_pages, const float* table, int64_t n_positions, int rot_dim, int offset,
           const int32_t* positions, int n_axes, const uint8_t* axes, int interleaved, void* k_codes, void* v_codes,
           float* k_scale, float* v_scale, sgl_stream_t stream) {
  SGL_REQUIRE(dtype == SGL_BF16 || dtype == SGL_F16 || dtype == SGL_F32, "kv8_append: dtype %d", dtype);
  const int rc = kv8_check_cache("kv8_append", Hkv, D, page_size, block, n_pages, row_pages);
  if (rc != SGL_OK) return rc;
  SGL_REQUIRE(T >= 0 && T <= (1 << 30) && B >= 0 && B <= (1 << 24), "kv8_append: T=%lld B=%lld out of range",
              (long long)T, (long long)B);
  SGL_REQUIRE(cu_tokens || T == B, "kv8_append: without cu_tokens every sequence has one token (T=%lld, B=%lld)",
              (long long)T, (long long)B);
  if (table) {
    SGL_REQUIRE(rot_dim >= 16 && rot_dim % 16 == 0 && offset >= 0 && offset % 8 == 0 && offset + rot_dim <= D,
                "kv8_append: rot_dim=%d must be a multiple of 16 and fit at offset %d (a multiple of 8) into D=%d",
                rot_dim, offset, D);
    SGL_REQUIRE(n_positions >= 1 && aligned(table, 16), "kv8_append: bad rotary table");
  }
  if (AXES) {
    SGL_REQUIRE(n_axes >= 1 && n_axes <= kMaxAxes, "kv8_append: n_axes=%d must be 1 to %d", n_axes, kMaxAxes);
    SGL_REQUIRE(n_positions <= 0x7FFFFFFF && n_positions * (rot_dim / 2) <= 0x7FFFFFFF,
                "kv8_append: a table of %lld positions is too large", (long long)n_positions);
  }
  if (T == 0 || B == 0) return SGL_OK;
  SGL_REQUIRE(k && v && start && block_table && k_codes && v_codes && k_scale && v_scale,
              "kv8_append: null pointer");
  SGL_REQUIRE(!AXES || (table && positions && axes), "kv8_append: axes need a table and positions");
  const int size = dtype == SGL_F32 ? 4 : 2;
  SGL_REQUIRE(aligned(k, 16) && aligned(v, 16) && k_token_stride * size % 16 == 0 &&
                  k_head_stride * size % 16 == 0 && v_token_stride * size % 16 == 0 && v_head_stride * size % 16 == 0,
              "kv8_append: k and v and their strides must be 16-byte aligned");
  SGL_REQUIRE(aligned(k_codes, 16) && aligned(v_codes, 16), "kv8_append: misaligned cache");
  AppendArgs a;
  a.k = k;
  a.v = v;
  a.kt = k_token_stride;
  a.kh = k_head_stride;
  a.vt = v_token_stride;
  a.vh = v_head_stride;
  a.kc = (uint8_t*)k_codes;
  a.vc = (uint8_t*)v_codes;
  a.ks = k_scale;
  a.vs = v_scale;
  a.pages = block_table;
  a.start = start;
  a.cu = cu_tokens;
  a.table = table;
  a.positions = positions;
  a.axes = axes;
  a.n_axes = n_axes;
  a.n_positions = n_positions;
  a.n_pages = n_pages;
  a.T = (int)T;
  a.B = (int)B;
  a.Hkv = Hkv;
  a.D = D;
  a.row_pages = (int)row_pages;
  a.page_shift = __builtin_ctz((unsigned)page_size);
  a.block_shift = __builtin_ctz((unsigned)block);
  a.per_magic = 65536 / (D / 16) + 1;
  a.rot = table ? rot_dim : 0;
  a.offset = table ? offset : 0;
  a.interleaved = interleaved != 0;
  const int64_t units = cu_tokens ? kv8_append_units(T, B, block) : B;
  const int64_t per_unit = (cu_tokens ? (int64_t)block : 1) * (D / 16);
  if (dtype == SGL_BF16)
    launch_append<SGL_BF16, AXES>(a, units, per_unit, (hipStream_t)stream);
  else if (dtype == SGL_F16)
    launch_append<SGL_F16, AXES>(a, units, per_unit, (hipStream_t)stream);
  else
    launch_append<SGL_F32, AXES>(a, units, per_unit, (hipStream_t)stream);
  return check_launch("kv8_append");
}

}  // namespace
}  // namespace sgl

extern "C" {

int sgl_kv8_append(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                   int64_t v_token_stride, int64_t v_head_stride, int dtype, int64_t T, int64_t B, int Hkv, int D,
                   const int32_t* cu_tokens, const int32_t* start, const int32_t* block_table, int64_t row_pages,
                   int page_size, int block, int64_t n_pages, const float* table, int64_t n_positions, int rot_dim,
                   int offset, const int32_t* positions, int interleaved, void* k_codes, void* v_codes,
                   float* k_scale, float* v_scale, sgl_stream_t stream) {
  return sgl::append<false>(k, k_token_stride, k_head_stride, v, v_token_stride, v_head_stride, dtype, T, B, Hkv, D,
                            cu_tokens, start, block_table, row_pages, page_size, block, n_pages, table, n_positions,
                            rot_dim, offset, positions, 1, nullptr, interleaved, k_codes, v_codes, k_scale, v_scale,
                            stream);
}

int sgl_kv8_append_axes(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                        int64_t v_token_stride, int64_t v_head_stride, int dtype, int64_t T, int64_t B, int Hkv, int D,
                        const int32_t* cu_tokens, const int32_t* start, const int32_t* block_table, int64_t row_pages,
                        int page_size, int block, int64_t n_pages, const float* table, int64_t n_positions,
                        int rot_dim, int offset, const int32_t* positions, int n_axes, const uint8_t* pair_axes,
                        int interleaved, void* k_codes, void* v_codes, float* k_scale, float* v_scale,
                        sgl_stream_t stream) {
  return sgl::append<true>(k, k_token_stride, k_head_stride, v, v_token_stride, v_head_stride, dtype, T, B, Hkv, D,
                           cu_tokens, start, block_table, row_pages, page_size, block, n_pages, table, n_positions,
                           rot_dim, offset, positions, n_axes, pair_axes, interleaved, k_codes, v_codes, k_scale,
                           v_scale, stream);
}

}  // extern "C"
