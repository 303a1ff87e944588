// Attention over the 8-bit paged cache: many rows a sequence and head (prompt
// chunks).  The mathematics, and the kernel for few rows: kv8_attn.hip.
//
// Bound by the matrix cores and, beside them, by the softmax's VALU work (an
// exponential is four issue slots).  Four wavefronts of 32 rows each share the
// key tiles of 64 tokens, whose codes are converted once, on the way into LDS
// (exact in bf16 and f16), and both products are v_mfma_f32_32x32x16:
//   S^T = K . Q^T (Q^T fragments stay in registers), O^T += V^T . P^T, where
//   P^T is the accumulator of S^T itself (its output layout is the B operand's)
//   and V^T comes from the row-major tile by ds_read_b64_tr_b16.
// Lane (row c, half g) owns row c in both: no exchange but the sum of two halves.
// S^T of tile j + 1 is computed beside the softmax of tile j: independent work
// that the scheduler lays between each other.  Codes are loaded two tiles ahead
// and stored one ahead; one barrier a tile.
#include "sgl_kv8_attn.h"

namespace sgl {
namespace {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef v4s __attribute__((address_space(3))) lds_v4s;
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

constexpr int kKeys = 64;  // tokens of a key tile

template <int QT>
struct Wide;
template <>
struct Wide<SGL_BF16> {
  static __device__ __forceinline__ v16f mfma(u4v a, u4v b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ __forceinline__ uint32_t cvt(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pk2_bf16(a, b); }
};
template <>
struct Wide<SGL_F16> {
  static __device__ __forceinline__ v16f mfma(u4v a, u4v b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ __forceinline__ uint32_t cvt(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack2<SGL_F16>(a, b); }
};

__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A row-major tile in LDS: token t, 16-byte chunk c at t ROW + ((c ^ swt(t)) << 4).
// Conflict-free for the fragment reads (one chunk of 16 consecutive tokens) and
// the transpose reads (four chunks of four consecutive tokens): rows of 16
// chunks and more rotate the token's low four bits; rows of 8 lie two to a
// 256-byte line, so the token's lowest bit already picks the half.
template <int DP>
__device__ __forceinline__ uint32_t swt(int t) {
  return DP >= 128 ? (uint32_t)(((t & 3) << 2) | ((t >> 2) & 3)) : (uint32_t)(((t & 2) << 1) | ((t >> 2) & 3));
}

// DP: head dim rounded up to 64, 128 or 256; NW wavefronts
template <int DP, int QT, int NW, bool SPLIT>
__global__ __launch_bounds__(64 * NW, DP == 256 ? 1 : 2) void kv8_prefill_kernel(const Kv8AttnArgs a, int64_t items) {
  constexpr int RT = 32 * NW, NT = 64 * NW, ROW = 2 * DP, KS = DP / 16, DT = DP / 32;
  constexpr int CPR = DP / 16;                  // 16-byte pieces of codes a token
  constexpr int PIECES = kKeys * CPR / NT;      // of a thread, for K and for V each
  constexpr int TSTEP = NT / CPR;               // tokens between a thread's pieces
  typedef Wide<QT> O;
  __shared__ __align__(16) uint8_t sK[2][kKeys * ROW];
  __shared__ __align__(16) uint8_t sV[2][kKeys * ROW];
  __shared__ __align__(4) uint16_t sDims[2][kKeys][CPR];  // of a tile seen in part: a token's dims with NaN codes
  __shared__ int sNan[2];                                 // 1 + the last such tile in the buffer that has any
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c32 = lane & 31, g2 = lane >> 5;
  const float NEG_INF = -__builtin_huge_valf();

  if (threadIdx.x < 2) sNan[threadIdx.x] = 0;
  int head, part = 0;
  Kv8Walk<RT, kKeys> walk;
  Kv8Segment seg;
  if constexpr (SPLIT) {
    kv8_wg_at(a, (int)blockIdx.x, &head, &part);
    if (!walk.start(a, part)) return;
  } else {
    // the last row tiles, which see the most keys, first; the heads go round
    // fastest, so that a head's workgroups meet on one XCD and its L2
    const int64_t item = items - 1 - (int64_t)blockIdx.x;
    head = (int)(item % a.Hkv);
    walk.c = kv8_chunk<RT, kKeys>(a, 0);
    const Kv8Place at = kv8_find<RT, kKeys, true>(a, walk.c, item / a.Hkv);
    if (at.l < 0) return;
    seg.s = kv8_lane<RT, kKeys>(a, walk.c, at.l);
    seg.b = walk.c.b0 + at.l;
    seg.rt = (int)(item / a.Hkv - at.rts);
    seg.t0 = 0;
    seg.t1 = seg.s.tiles;
  }
  for (bool more = SPLIT ? walk.next(a, seg) : true; more; more = SPLIT ? walk.next(a, seg) : false) {
    const Kv8Seq& s = seg.s;
    const int b = seg.b, rt = seg.rt, t0 = seg.t0, t1 = seg.t1;
    const int rows = s.n * a.G - rt * RT;
    const bool whole = t0 == 0 && t1 == s.tiles;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (t0 == 0 ? 1 : 0);

    // this lane's row, and what it sees
    const int r = 32 * wave + c32;
    const bool live = r < rows;
    const int row = rt * RT + (live ? r : 0), tq = row / a.G, hq = head * a.G + (row - tq * a.G);
    const int pos = s.len - s.n + tq;
    const int hi = !live ? 0 : a.causal && pos + 1 < s.len ? pos + 1 : s.len;
    const int lo = a.causal && a.window > 0 ? pos - a.window + 1 : 0;
    // what all rows of the wavefront see, and what any row of the tile sees
    int all_hi = s.len, all_lo = 0, any_lo = 0, any_hi = s.len;
    if (a.causal) {
      const int first = rt * RT, last = first + (rows < RT ? rows : RT) - 1;
      const int w0 = first + 32 * wave, w1 = w0 + 31 < last ? w0 + 31 : last;
      all_hi = s.len - s.n + w0 / a.G + 1;
      all_hi = all_hi < s.len ? all_hi : s.len;
      any_hi = s.len - s.n + last / a.G + 1;
      if (a.window > 0) {
        all_lo = s.len - s.n + w1 / a.G - a.window + 1;
        any_lo = s.len - s.n + first / a.G - a.window + 1;
        any_lo = any_lo < 0 ? 0 : any_lo;
      }
    }
    int j0 = s.tile0 + t0, j1 = s.tile0 + t1;
    if (any_lo / kKeys > j0) j0 = any_lo / kKeys;
    const int jh = any_hi <= 0 ? 0 : (any_hi + kKeys - 1) / kKeys;
    if (jh < j1) j1 = jh;
    if (s.len == 0) j1 = j0;

    v16f acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
    float m_run = NEG_INF, l_run = 0.0f;

    if (j0 < j1) {
      u4v q[KS];
      {
        const uint16_t* src = a.q + (int64_t)(s.row0 + tq) * a.qt + (int64_t)hq * a.qh + 8 * g2;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          q[k] = u4v{0, 0, 0, 0};
          if (live && 16 * k < a.D) q[k] = *reinterpret_cast<const u4v*>(src + 16 * k);
        }
      }
      const int32_t* table = a.pages + (int64_t)b * a.row_pages;
      const int pmask = (1 << a.page_shift) - 1;
      const int last_tok = s.len - 1;

      // ---- staging: piece i of this thread is 16 codes of token ptok + i TSTEP
      const int pc = threadIdx.x % CPR, ptok = threadIdx.x / CPR;
      const bool in_d = 16 * pc < a.D;
      struct Pages {
        int p[PIECES];
      };
      auto load_pages = [&](int j) {
        Pages o;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          int t = j * kKeys + ptok + i * TSTEP;
          t = t < s.len ? t : last_tok;
          o.p[i] = table[t >> a.page_shift];
        }
        return o;
      };
      auto load_codes = [&](const uint8_t* codes, int j, const Pages& pg, uint4* out) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          int t = j * kKeys + ptok + i * TSTEP;
          const bool ok = t < s.len && pg.p[i] >= 0 && pg.p[i] < a.n_pages && in_d;
          t = t < s.len ? t : last_tok;
          const int64_t line = (int64_t)(ok ? pg.p[i] : 0) * a.Hkv + head;
          out[i] = make_uint4(0, 0, 0, 0);
          if (ok)
            out[i] = *reinterpret_cast<const uint4*>(codes + ((line << a.page_shift) + (t & pmask)) * a.D + 16 * pc);
        }
      };
      auto store_codes = [&](uint8_t* tile, const uint4* in) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int t = ptok + i * TSTEP;
          const uint32_t w[4] = {in[i].x, in[i].y, in[i].z, in[i].w};
          u4v lo, hi2;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            lo[2 * k] = O::template cvt<false>(w[k]);
            lo[2 * k + 1] = O::template cvt<true>(w[k]);
            hi2[2 * k] = O::template cvt<false>(w[2 + k]);
            hi2[2 * k + 1] = O::template cvt<true>(w[2 + k]);
          }
          *reinterpret_cast<u4v*>(tile + t * ROW + (((2 * pc) ^ swt<DP>(t)) << 4)) = lo;
          *reinterpret_cast<u4v*>(tile + t * ROW + (((2 * pc + 1) ^ swt<DP>(t)) << 4)) = hi2;
        }
      };
      // A tile that some rows see in part: its NaN codes are zeroed, so that 0 * NaN
      // reaches no row's sum, and noted, for the rows that do see them.
      auto take_nan = [&](int j, uint4* in) {
        bool any = false;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          uint32_t w[4] = {in[i].x, in[i].y, in[i].z, in[i].w}, dims = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t bad = (((w[k] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;  // 1 in a NaN's byte
            w[k] &= ~(bad * 0xFFu);
            dims |= ((bad * 0x10204080u) >> 28) << (4 * k);
          }
          in[i] = make_uint4(w[0], w[1], w[2], w[3]);
          sDims[j & 1][ptok + i * TSTEP][pc] = (uint16_t)dims;
          any |= dims != 0;
        }
        if (any) sNan[j & 1] = j + 1;
      };
      const int part_hi = a.causal ? s.len - s.n + (rt * RT) / a.G + 1 : s.len;  // keys that the first row sees
      const int part_lo = a.causal && a.window > 0
                              ? s.len - s.n + (rt * RT + (rows < RT ? rows : RT) - 1) / a.G - a.window + 1 : 0;
      auto partial = [&](int j) { return (j + 1) * kKeys > part_hi || j * kKeys < part_lo; };

      // ---- scales: lane i < 4 has granule i of a tile
      struct Scales {
        float k, v;
        bool ok;
      };
      auto load_scales = [&](int j) {
        Scales o;
        const int t = j * kKeys + 16 * (lane & 3);
        const int u = t < s.len ? t : last_tok & ~15;
        const int page = table[u >> a.page_shift];
        o.ok = page >= 0 && page < a.n_pages && t < s.len;
        const int64_t line = (int64_t)(o.ok ? page : 0) * a.Hkv + head;
        const int64_t piece = (line << (a.page_shift - a.block_shift)) + ((u & pmask) >> a.block_shift);
        o.k = a.ks[piece];
        o.v = a.vs[piece];
        return o;
      };

      // ---- S^T of tile j: lane (row c32, half g2) gets token 32 t + 8 (i / 4) + 4 g2 + i % 4 in sc[t][i]
      uint32_t ka[DP >= 128 ? 8 : 4];
#pragma unroll
      for (int k = 0; k < (DP >= 128 ? 8 : 4); ++k)
        ka[k] = c32 * ROW + (((2 * k + g2) ^ swt<DP>(c32)) << 4);
      auto scores = [&](int j, v16f* sc) {
        const uint8_t* tile = sK[j & 1];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[t][i] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < KS; ++k) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const u4v kf = *reinterpret_cast<const u4v*>(tile + ka[k & 7] + 32 * t * ROW + 256 * (k >> 3));
            sc[t] = O::mfma(kf, q[k], sc[t]);
          }
        }
      };
      uint32_t va[2][DT > 4 ? 4 : DT];
      {
        const int G = lane >> 4, s16 = lane & 15;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int d = 0; d < (DT > 4 ? 4 : DT); ++d) {
            const int tok = 8 * e + 4 * (G >> 1) + (s16 >> 2);
            const int ch = 4 * d + 2 * (G & 1) + ((s16 & 3) >> 1);
            va[e][d] = tok * ROW + ((ch ^ swt<DP>(tok)) << 4) + 8 * (s16 & 1);
          }
      }
      auto v_frag = [&](const uint8_t* tile, int s4, int d) {
        const v4s l = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_v4s*)(tile + va[0][d & 3] + 256 * (d >> 2) + 16 * s4 * ROW));
        const v4s h = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_v4s*)(tile + va[1][d & 3] + 256 * (d >> 2) + 16 * s4 * ROW));
        return __builtin_bit_cast(u4v, __builtin_shufflevector(l, h, 0, 1, 2, 3, 4, 5, 6, 7));
      };

      // ---- one tile: softmax of sc (tile j), S^T of tile j + 1 into sn, O^T += V^T . P^T
      uint4 rk[PIECES], rv[PIECES];
      Pages pk, pv;
      Scales sj, sj1;
      auto tile_step = [&](int j, v16f* sc, v16f* sn) {
        store_codes(sK[j & 1], rk);                // tile j + 2
        if (partial(j + 1)) take_nan(j + 1, rv);
        store_codes(sV[(j + 1) & 1], rv);          // tile j + 1
        load_codes(a.kc, j + 3, pk, rk);
        load_codes(a.vc, j + 2, pv, rv);
        pv = pk;
        pk = load_pages(j + 4);
        // P^T = 2^(s + log2 s_v - m), so that s_v is in the exponent, and the sum takes it back
        const float kc = sj.ok ? sj.k * a.c1 : 0.0f;
        const float e = sj.ok ? __builtin_fmaxf(__builtin_amdgcn_logf(sj.v), -100.0f) : 0.0f;
        const float iv = __builtin_amdgcn_exp2f(-e);
        const uint64_t okm = __ballot(sj.ok);
        sj = sj1;
        sj1 = load_scales(j + 2);
        scores(j + 1, sn);
        const int tok = j * kKeys;
        const bool plain = tok + kKeys <= all_hi && tok >= all_lo && (okm & 15) == 15;
        float mx = NEG_INF;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float kg = bits_f32(__builtin_amdgcn_readlane(f32_bits(kc), g));
          const float eg = bits_f32(__builtin_amdgcn_readlane(f32_bits(e), g));
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = 8 * (g & 1) + i;
            sc[g >> 1][at] = __builtin_fmaf(sc[g >> 1][at], kg, eg);
          }
        }
        if (!plain) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int key = tok + 32 * t + 8 * (i >> 2) + 4 * g2 + (i & 3);
              if (!(key < hi && key >= lo && ((okm >> (2 * t + (i >> 3))) & 1))) sc[t][i] = NEG_INF;
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = __builtin_fmaxf(mx, sc[t][i]);
        // the reference moves only when a score exceeds it by more than 6 (log2
        // units): the weights stay at most 64, the accumulators are rarely rescaled
        if (__ballot(!(mx <= m_run + 6.0f) && mx != NEG_INF)) {
          mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32, 64));
          const float nx = mx <= m_run + 6.0f ? m_run : __builtin_fmaxf(m_run, mx);
          const float alpha = nx == m_run ? 1.0f : __builtin_amdgcn_exp2f(m_run - nx);
          m_run = nx;
          l_run *= alpha;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[d][i] *= alpha;
        }
        const float ref = m_run == NEG_INF ? 0.0f : m_run;
        u4v p[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float ig = bits_f32(__builtin_amdgcn_readlane(f32_bits(iv), g));
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const float u = __builtin_amdgcn_exp2f(sc[g >> 1][8 * (g & 1) + i] - ref);
            const float w = __builtin_amdgcn_exp2f(sc[g >> 1][8 * (g & 1) + i + 1] - ref);
            sum += u;
            sum += w;
            p[g][i >> 1] = O::pack(u, w);
          }
          l_run = __builtin_fmaf(sum, ig, l_run);
        }
        const uint8_t* tile = sV[j & 1];
#pragma unroll
        for (int s4 = 0; s4 < 4; ++s4)
#pragma unroll
          for (int d = 0; d < DT; ++d) acc[d] = O::mfma(v_frag(tile, s4, d), p[s4], acc[d]);
        if (partial(j) && sNan[j & 1] == j + 1) {
          for (int t = 0; t < kKeys; ++t) {
            const bool seen = tok + t < hi && tok + t >= lo;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              const uint32_t dims = *reinterpret_cast<const uint32_t*>(&sDims[j & 1][t][2 * d]) >> (4 * g2);
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (seen && ((dims >> (8 * (i >> 2) + (i & 3))) & 1u)) acc[d][i] = __builtin_nanf("");
            }
          }
        }
        lds_barrier();
      };

      // ---- tiles j0, j0 + 1 into LDS, S^T of the first
      lds_barrier();  // the last segment's reads, and sNan
      {
        const Pages p0 = load_pages(j0), p1 = load_pages(j0 + 1), p2 = load_pages(j0 + 2);
        sj = load_scales(j0);
        sj1 = load_scales(j0 + 1);
        uint4 r1[PIECES];
        load_codes(a.kc, j0, p0, rk);
        load_codes(a.vc, j0, p0, rv);
        load_codes(a.kc, j0 + 1, p1, r1);
        pk = load_pages(j0 + 3);
        store_codes(sK[j0 & 1], rk);
        store_codes(sK[(j0 + 1) & 1], r1);
        if (partial(j0)) take_nan(j0, rv);
        store_codes(sV[j0 & 1], rv);
        load_codes(a.kc, j0 + 2, p2, rk);
        load_codes(a.vc, j0 + 1, p1, rv);
        pv = p2;
      }
      lds_barrier();
      v16f s0[2], s1[2];
      scores(j0, s0);
      lds_barrier();
      for (int j = j0; j < j1; j += 2) {
        tile_step(j, s0, s1);
        if (j + 1 >= j1) break;
        tile_step(j + 1, s1, s0);
      }
    }

    // ---- out
    l_run += __shfl_xor(l_run, 32, 64);
    if (live) {
      if (whole) {
        const float ref = m_run == NEG_INF ? 0.0f : m_run;
        const float sum = a.sink ? l_run + __builtin_amdgcn_exp2f(a.sink[hq] * kLog2e - ref) : l_run;
        const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
        uint16_t* o = a.o + ((int64_t)(s.row0 + tq) * (a.Hkv * a.G) + hq) * a.D + 4 * g2;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (32 * d + 8 * k < a.D)
              *reinterpret_cast<uint2*>(o + 32 * d + 8 * k) =
                  make_uint2(kv8_out2<QT>(acc[d][4 * k] * inv, acc[d][4 * k + 1] * inv),
                             kv8_out2<QT>(acc[d][4 * k + 2] * inv, acc[d][4 * k + 3] * inv));
      } else {
        float* o = a.ws_acc + (slot * RT + r) * a.D + 4 * g2;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (32 * d + 8 * k < a.D)
              *reinterpret_cast<float4*>(o + 32 * d + 8 * k) =
                  make_float4(acc[d][4 * k], acc[d][4 * k + 1], acc[d][4 * k + 2], acc[d][4 * k + 3]);
        if (g2 == 0) *reinterpret_cast<float2*>(a.ws_ml + (slot * RT + r) * 2) = make_float2(m_run, l_run);
      }
    }
  }
}

template <int DP, int QT>
void launch_prefill(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t st) {
  const int64_t items = kv8_attn_items(a.T, a.B, a.Hkv, a.G, 128);
  if (p.parts == 0) {
    kv8_prefill_kernel<DP, QT, 4, false><<<(unsigned)items, 256, 0, st>>>(a, items);
  } else {
    kv8_prefill_kernel<DP, QT, 4, true><<<a.parts * a.Hkv, 256, 0, st>>>(a, items);
    kv8_merge_kernel<128, kKeys, QT><<<(unsigned)(items * 32), 256, 0, st>>>(a);
  }
}

template <int QT>
void launch_prefill_as(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t st) {
  if (a.D <= 64)
    launch_prefill<64, QT>(a, p, st);
  else if (a.D <= 128)
    launch_prefill<128, QT>(a, p, st);
  else
    launch_prefill<256, QT>(a, p, st);
}

}  // namespace

void launch_kv8_prefill(const Kv8AttnArgs& a, const Kv8AttnPlan& p, int dtype, hipStream_t st) {
  if (dtype == SGL_BF16)
    launch_prefill_as<SGL_BF16>(a, p, st);
  else
    launch_prefill_as<SGL_F16>(a, p, st);
}

}  // namespace sgl
