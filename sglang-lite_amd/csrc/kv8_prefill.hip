// Attention over the 8-bit paged cache: many rows a sequence and head (prompt
// chunks).  The mathematics, and the kernel for few rows: kv8_attn.hip.
//
// Bound by the matrix cores and, beside them, the softmax's VALU work (8192 queries
// of 32 heads of 128 on 8 kv heads: 550 to 564 us, 0.98 to 1.0 PFLOP/s; MFMA 47 %, VALU 45 % busy).
// Eight wavefronts (heads up to 64 and above 128: four) of 32 rows each share the key
// tiles of 64 tokens (heads above 128: 32), whose codes are converted once, on the
// way into LDS (exact in bf16 and f16), and both products are v_mfma_f32_32x32x16:
//   S^T = K . Q^T (Q^T fragments in registers, or LDS for wide heads), O^T += V^T . P^T, where
//   P^T is the accumulator of S^T itself (its output layout is the B operand's)
//   and V^T comes from the row-major tile by ds_read_b64_tr_b16.
// Lane (row c, half g) owns row c in both: no exchange but the sum of two halves.
// The softmax of tile j lies, a pair of weights at a time, between the products
// S^T of tile j + 1 and O^T of tile j - 1: VALU instructions of the same wavefront
// run in an MFMA's shadow (32 cycles: four of them for nothing, eight for half),
// those of another wavefront's softmax phase much less.  One barrier a tile.
// Wavefronts of 64 rows halve the LDS reads, but not the time: 690 us with tiles of 32
// tokens, 830 with 64, which spill.  Heads of 256, 4096 queries of 16 heads: 214 us
// (MFMA 28 %, VALU 26 %, LDS 36 %: one wavefront a SIMD waits for itself); 612 with tiles of
// 64 tokens and Q in registers, which spill.
#include "sgl_kv8_attn.h"

namespace sgl {
namespace {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef v4s __attribute__((address_space(3))) lds_v4s;
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

// Tokens of a key tile: 64; 32 of heads above 128, whose accumulators leave less room.
constexpr int chunk_keys(int DP) { return DP == 256 ? 32 : 64; }

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
// V's tile is read by the transpose alone and rotates two bits, so that its reads 8
// tokens on differ by a constant.
template <int DP>
__device__ __forceinline__ uint32_t swv(int t) {
  return DP >= 128 ? (uint32_t)((t & 3) << 2) : (uint32_t)((t & 2) << 1);
}
template <int DP>
__device__ __forceinline__ uint32_t swt(int t) {
  return DP >= 128 ? (uint32_t)(((t & 3) << 2) | ((t >> 2) & 3)) : (uint32_t)(((t & 2) << 1) | ((t >> 2) & 3));
}

// DP: head dim rounded up to 64, 128 or 256; NW wavefronts
template <int DP, int QT, int NW, bool SPLIT, int MODE>
__global__ __launch_bounds__(64 * NW, DP == 256 ? 1 : 2) void kv8_prefill_kernel(const Kv8AttnArgs a, int64_t items) {
  constexpr bool FIRST = MODE == kFirst;
  constexpr int kKeys = chunk_keys(DP), NG = kKeys / 16, NH = kKeys / 32;  // granules, halves of 32 tokens
  constexpr int RT = 32 * NW, NT = 64 * NW, ROW = 2 * DP, KS = DP / 16, DT = DP / 32;
  constexpr int NS = KS * NH;   // products of each kind in a tile
  constexpr int TB = 64 / NG;   // tiles whose granules' scales and pages the lanes hold
  static_assert(NS == NG * DT, "as many of S as of O");
  constexpr int CPR = DP / 16;               // 16-byte pieces of codes a token
  constexpr int SIDE = kKeys * CPR;          // pieces of K's tile, and of V's behind them
  constexpr int PIECES = 2 * SIDE / NT;      // of a thread
  static_assert(PIECES * NT == 2 * SIDE && SIDE % NT == 0, "a thread's first pieces are K's, the others V's");
  typedef Wide<QT> O;       // K's codes, as q
  typedef Wide<SGL_F16> F;  // V's codes and the weights
  __shared__ __align__(16) uint8_t sK[4][kKeys * ROW];  // K, K, V, V
  // Q^T fragments: in LDS where the registers are short
  constexpr bool QL = DP >= 128;
  __shared__ __align__(16) u4v sQ[QL ? NW : 1][QL ? KS : 1][64];
  __shared__ __align__(4) uint16_t sDims[2][kKeys][CPR];  // of a tile seen in part: a token's dims with NaN codes
  __shared__ __align__(8) float2 sScale[2][64];           // of a batch's granules: score scale, kLift + log2 of the value scale
  __shared__ int sNan[2];                                 // 1 + the last such tile in the buffer that has any
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c32 = lane & 31, g2 = lane >> 5;
  const float NEG_INF = -__builtin_huge_valf();

  if (threadIdx.x < 2) sNan[threadIdx.x] = 0;
  int head, part = 0;
  Kv8Walk<RT, kKeys, MODE> walk;
  Kv8Segment seg;
  if constexpr (SPLIT) {
    kv8_wg_at(a, (int)blockIdx.x, &head, &part);
    if (!walk.start(a, part)) return;
  } else {
    // the last row tiles, which see the most keys, first; the heads go round
    // fastest, so that a head's workgroups meet on one XCD and its L2
    if (!kv8_item<RT, kKeys, MODE>(a, items - 1 - (int64_t)blockIdx.x, &head, seg)) return;
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
    // (without branches, and the masks below too, which choose an element's value and always store it.  Where
    // lanes part and come together around the store of one element of a vector, the compiler (ROCm 7.2)
    // may empty the block that stores: it made that of `key < hi && (key >= lo || key < first)`, and keys that the
    // window hides were seen.)
    const uint32_t hidden = lo > a.first ? (uint32_t)(lo - a.first) : 0u;  // keys between the first tokens and the window
    auto sees = [&](int key) __attribute__((always_inline)) {
      if constexpr (FIRST)
        return (key < hi) & ((uint32_t)(key - a.first) >= hidden);
      else
        return (key < hi) & (key >= lo);
    };
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
    // The tiles to go over: of the first tokens those from t0 on, `front` of them, then
    // from j0 on, where the windows of these rows begin.
    int front = 0, j0 = t0, j1 = s.tile0 + t1;
    const int jh = any_hi <= 0 ? 0 : (any_hi + kKeys - 1) / kKeys;
    if (FIRST && t0 < s.kept) {
      front = (t1 < s.kept ? t1 : s.kept) < jh ? (t1 < s.kept ? t1 : s.kept) - t0 : jh - t0;
      front = front > 0 ? front : 0;
      if (t1 <= s.kept) j1 = 0;  // (nothing behind them)
      j0 = s.kept;
    }
    j0 += s.tile0;
    if (any_lo / kKeys > j0) j0 = any_lo / kKeys;
    if (jh < j1) j1 = jh;
    const int n_tiles = s.len == 0 ? 0 : front + (j1 > j0 ? j1 - j0 : 0);
    auto tile_at = [&](int i) __attribute__((always_inline)) { return FIRST && i < front ? t0 + i : i + (FIRST ? j0 - front : j0); };

    v16f acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
    float m_run = live ? NEG_INF : 1e30f, l_run = 0.0f;  // (a row that is none never asks for a reference)

    if (n_tiles > 0) {
      u4v q[KS];  // (with QL only until they are in LDS)
      {
        const uint16_t* src = a.q + (int64_t)(s.row0 + tq) * a.qt + (int64_t)hq * a.qh + 8 * g2;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          q[k] = u4v{0, 0, 0, 0};
          if (live && 16 * k < a.D) q[k] = *reinterpret_cast<const u4v*>(src + 16 * k);
        }
      }
      auto q_frag = [&](int k) __attribute__((always_inline)) {
        if constexpr (QL)
          return sQ[wave][k][lane];
        else
          return q[k];
      };
      const int32_t* table = a.pages + (int64_t)(MODE == kShared && a.table_row ? a.table_row[b] : b) * a.row_pages;
      const int pmask = (1 << a.page_shift) - 1;

      // ---- pages and scales of TB tiles at a time: lane l has granule l % NG of tile
      // l / NG, in their order; pages loaded a batch ahead, scales most of one
      struct Batch {
        int page;  // 0 where there is none
        float k, v;
        bool ok;  // the granule lies before the end, on a page of the cache
      };
      auto load_pages = [&](int batch) __attribute__((always_inline)) {
        Batch o;
        const int t = tile_at(TB * batch + lane / NG) * kKeys + 16 * (lane % NG);
        const int page = table[(t < s.len ? t : s.len - 1) >> a.page_shift];
        o.ok = t < s.len && page >= 0 && page < a.n_pages;
        o.page = o.ok ? page : 0;
        return o;
      };
      auto load_scales = [&](int batch, Batch& o) __attribute__((always_inline)) {
        const int t = tile_at(TB * batch + lane / NG) * kKeys + 16 * (lane % NG);
        const int64_t piece = (((int64_t)o.page * a.Hkv + head) << (a.page_shift - a.block_shift)) +
                              ((t & pmask) >> a.block_shift);
        o.k = a.ks[piece];
        o.v = a.vs[piece];
      };
      // A granule's two numbers are read back as a broadcast (v_readlane takes four
      // times as long as a plain VALU instruction here).  Every wavefront writes the
      // same values to the same place, and reads behind its own writes.
      uint64_t okm = 0;  // granules that are there, with scales as they should be
      auto use = [&](int batch, const Batch& o) __attribute__((always_inline)) {
        // (what was never written may hold anything).  A score of -inf, a key not seen,
        // has to stay one: a scale of 0 becomes the smallest above it.
        const bool good = kv8_scale_ok(o.k) && kv8_scale_ok(o.v);
        const float k = o.k * a.c1;
        sScale[batch & 1][lane] =
            make_float2(!o.ok || !good ? 1.0f : k == 0.0f ? 0x1p-149f : k, kv8_exponent(o.ok, good, o.v));
        okm = __ballot(o.ok && good && o.v >= 0x1p-100f);
      };

      // ---- staging: piece i of this thread is 16 codes of token ptok + i TSTEP.  A
      // wavefront's piece lies in one granule, so its page is one number.
      const int pc = threadIdx.x % CPR, ptok = threadIdx.x / CPR;
      const int wtok = wave * (64 / CPR);
      const uint32_t poff = (uint32_t)((ptok - wtok) * a.D + (16 * pc < a.D ? 16 * pc : 0));
      // piece i: whether V's, and its token (the wavefront's first: with wtok)
      auto is_v = [](int i) { return i * NT >= SIDE; };
      auto tok_of = [&](int i, int t) { return (t + i * (NT / CPR)) % kKeys; };
      // K's pieces of the ik-th tile, V's of the iv-th (pages: the lanes' pages of their batches)
      auto load_codes = [&](int ik, int kpages, int iv, int vpages, uint4* out) __attribute__((always_inline)) {
        const int jk = tile_at(ik), jv = tile_at(iv);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int t = tok_of(i, wtok), j = is_v(i) ? jv : jk;
          const int page = __builtin_amdgcn_readlane(is_v(i) ? vpages : kpages, NG * ((is_v(i) ? iv : ik) & (TB - 1)) + (t >> 4));
          const int64_t row = (((int64_t)page * a.Hkv + head) << a.page_shift) + ((j * kKeys + t) & pmask);
          out[i] = *reinterpret_cast<const uint4*>((is_v(i) ? a.vc : a.kc) + row * a.D + poff);
        }
      };
      // (the swizzle repeats every 16 tokens: the same for all of a thread's pieces)
      static_assert(NT / CPR % 16 == 0, "tokens between a thread's pieces");
      auto dst = [&](int i, int half) {
        return ptok % kKeys * ROW + (((2 * pc + half) ^ (is_v(i) ? swv<DP>(ptok) : swt<DP>(ptok))) << 4);
      };
      const uint32_t kdst0 = dst(0, 0), kdst1 = dst(0, 1), vdst0 = dst(PIECES - 1, 0), vdst1 = dst(PIECES - 1, 1);
      auto store_piece = [&](int i, int buf, const uint4& in) __attribute__((always_inline)) {
        const uint32_t w[4] = {in.x, in.y, in.z, in.w};
        u4v lo, hi2;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          lo[2 * k] = is_v(i) ? F::template cvt<false>(w[k]) : O::template cvt<false>(w[k]);
          lo[2 * k + 1] = is_v(i) ? F::template cvt<true>(w[k]) : O::template cvt<true>(w[k]);
          hi2[2 * k] = is_v(i) ? F::template cvt<false>(w[2 + k]) : O::template cvt<false>(w[2 + k]);
          hi2[2 * k + 1] = is_v(i) ? F::template cvt<true>(w[2 + k]) : O::template cvt<true>(w[2 + k]);
        }
        uint8_t* to = sK[buf] + i * NT / SIDE * (2 * kKeys * ROW) + i * NT % SIDE / CPR * ROW;
        *reinterpret_cast<u4v*>(to + (is_v(i) ? vdst0 : kdst0)) = lo;
        *reinterpret_cast<u4v*>(to + (is_v(i) ? vdst1 : kdst1)) = hi2;
      };
      // Values behind the last key, or on no page, were never written: zeros, which
      // meet zeros of P.
      auto clear_missing = [&](int j, uint32_t here, uint4* in) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int t = tok_of(i, ptok);
          if (is_v(i) && (j * kKeys + t >= s.len || !((here >> (t >> 4)) & 1u))) in[i] = make_uint4(0, 0, 0, 0);
        }
      };
      // Values that count as zero: only NaN codes are left of them.
      auto clear_values = [&](uint32_t none, uint4* in) __attribute__((always_inline)) {
        auto nan_alone = [](uint32_t w) {
          return w & ((((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xFFu;
        };
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
          if (is_v(i) && ((none >> (tok_of(i, ptok) >> 4)) & 1u))
            in[i] = make_uint4(nan_alone(in[i].x), nan_alone(in[i].y), nan_alone(in[i].z), nan_alone(in[i].w));
      };
      // A tile that some rows see in part: its NaN codes are zeroed, so that 0 * NaN
      // reaches no row's sum, and noted, for the rows that do see them.
      auto take_nan = [&](int j, int buf, uint4* in) __attribute__((always_inline)) {
        bool any = false;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          if (!is_v(i)) continue;
          uint32_t w[4] = {in[i].x, in[i].y, in[i].z, in[i].w}, dims = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t bad = (((w[k] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;  // 1 in a NaN's byte
            w[k] &= ~(bad * 0xFFu);
            dims |= ((bad * 0x10204080u) >> 28) << (4 * k);
          }
          in[i] = make_uint4(w[0], w[1], w[2], w[3]);
          sDims[buf][tok_of(i, ptok)][pc] = (uint16_t)dims;
          any |= dims != 0;
        }
        if (any) sNan[buf] = j + 1;
      };
      const int part_hi = a.causal ? s.len - s.n + (rt * RT) / a.G + 1 : s.len;  // keys that the first row sees
      const int part_lo = a.causal && a.window > 0
                              ? s.len - s.n + (rt * RT + (rows < RT ? rows : RT) - 1) / a.G - a.window + 1 : 0;
      auto partial = [&](int j) {
        return (j + 1) * kKeys > part_hi || (j * kKeys < part_lo && !(FIRST && (j + 1) * kKeys <= a.first));
      };
      // ---- S^T: lane (row c32, half g2) gets token 32 t + 8 (i / 4) + 4 g2 + i % 4 in sc[t][i]
      constexpr int NKA = DP >= 128 ? 8 : 4;
      uint32_t ka[NKA];
#pragma unroll
      for (int k = 0; k < NKA; ++k) ka[k] = c32 * ROW + (((2 * k + g2) ^ swt<DP>(c32)) << 4);
      constexpr int NVA = DT > 4 ? 4 : DT;
      uint32_t va[NVA];
      {
        const int G = lane >> 4, s16 = lane & 15;
#pragma unroll
        for (int d = 0; d < NVA; ++d) {
          const int tok = 4 * (G >> 1) + (s16 >> 2);
          const int ch = 4 * d + 2 * (G & 1) + ((s16 & 3) >> 1);
          va[d] = tok * ROW + ((ch ^ swv<DP>(tok)) << 4) + 8 * (s16 & 1);
        }
      }
      auto v_frag = [&](const uint8_t* tile, int s4, int d) __attribute__((always_inline)) {
        const v4s l = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_v4s*)(tile + va[d & 3] + 256 * (d >> 2) + 16 * s4 * ROW));
        const v4s h = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_v4s*)(tile + va[d & 3] + 256 * (d >> 2) + (16 * s4 + 8) * ROW));
        return __builtin_bit_cast(u4v, __builtin_shufflevector(l, h, 0, 1, 2, 3, 4, 5, 6, 7));
      };

      // NaN codes of tile j, for the rows that see them
      auto put_nan = [&](int j, int buf) __attribute__((always_inline)) {
        if (__builtin_expect(partial(j) && sNan[buf] == j + 1, 0)) {
          for (int t = 0; t < kKeys; ++t) {
            const bool seen = sees(j * kKeys + t);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              const uint32_t dims = *reinterpret_cast<const uint32_t*>(&sDims[buf][t][2 * d]) >> (4 * g2);
#pragma unroll
              for (int i = 0; i < 16; ++i)
                acc[d][i] = (seen & (((dims >> (8 * (i >> 2) + (i & 3))) & 1u) != 0)) ? __builtin_nanf("") : acc[d][i];
            }
          }
        }
      };
      auto k_frag = [&](const uint8_t* kt, int n) __attribute__((always_inline)) {
        const int k = n / NH, t = n % NH;
        return *reinterpret_cast<const u4v*>(kt + ka[k & 7] + 32 * t * ROW + 256 * (k >> 3));
      };

      uint4 raw[PIECES];  // K's codes of tile j + 2, V's of tile j
      u4v p[NG];          // P^T of tile j - 1
      constexpr uint32_t kAll = (1u << NG) - 1;
      bool fresh = __ballot(m_run == NEG_INF) != 0;  // a row has no reference yet
      Batch now, ahead;
      // The i-th tile j, scores in sc: its softmax, slice by slice between the products
      // S^T of tile j + 1 (into sn) and O^T += V^T . P^T of tile j - 1.
      auto tile_step = [&](int i, const int buf, v16f* sc, v16f* sn) __attribute__((always_inline)) {
        const int j = tile_at(i), l0 = NG * (i & (TB - 1)), tok = j * kKeys;
        const float2* scale = &sScale[(i / TB) & 1][l0];
        auto top = [&]() __attribute__((always_inline)) {  // the row's largest exponent in this tile
          float mx = NEG_INF;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            float mg = sc[g >> 1][8 * (g & 1)];
#pragma unroll
            for (int e = 1; e < 8; ++e) mg = __builtin_fmaxf(mg, sc[g >> 1][8 * (g & 1) + e]);
            mx = __builtin_fmaxf(mx, __builtin_fmaf(mg, scale[g].x, scale[g].y));
          }
          return __builtin_fmaxf(mx, __shfl_xor(mx, 32, 64));
        };
        // Everything that most tiles do not need stands behind one branch (a taken
        // branch costs a wavefront some 50 cycles): batch borders, the end of the keys,
        // masks, NaN codes, rows without a reference.
        // The reference m need not be the maximum: any m gives the same softmax.  So
        // no maximum is taken unless a row has no reference yet (its sums are zero
        // then), or, below, eight weights pass what one f16 holds.  It lies kLift
        // below the maximum that it was taken from.
        const bool border = (i & (TB - 1)) == 0 && i > 0;
        const bool seen_by_all = tok + kKeys <= all_hi && (tok >= all_lo || (FIRST && tok + kKeys <= a.first));
        if (__builtin_expect(border || (i & (TB - 1)) == 4 || !seen_by_all || partial(j) || (okm >> l0 & kAll) != kAll || fresh, 0)) {
          if (border) {
            now = ahead;
            use(i / TB, now);
            ahead = load_pages(i / TB + 1);
          }
          if ((i & (TB - 1)) == 4) load_scales(i / TB + 1, ahead);
          const uint32_t ok = (uint32_t)(okm >> l0) & kAll;
          uint32_t here = kAll;
          if (__builtin_expect(ok != kAll, 0)) {
            const float mark = sScale[(i / TB) & 1][lane].y;
            here = (uint32_t)(__ballot(mark != kNoToken) >> l0) & kAll;
            if (here != ok) {
              const uint32_t bad = (uint32_t)(__ballot(mark == kBadScale) >> l0);
#pragma unroll
              for (int t = 0; t < NH; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  sc[t][e] = (bad >> (2 * t + (e >> 3))) & 1 ? __builtin_nanf("") : sc[t][e];
              clear_values((uint32_t)(__ballot(mark == kNoValue) >> l0), raw);
            }
          }
          if (tok + kKeys > s.len || here != kAll) clear_missing(j, here, raw);
          if (partial(j)) take_nan(j, buf, raw);
          if (!seen_by_all || here != kAll) {
#pragma unroll
            for (int t = 0; t < NH; ++t)
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const int key = tok + 32 * t + 8 * (e >> 2) + 4 * g2 + (e & 3);
                sc[t][e] = (sees(key) & (((here >> (2 * t + (e >> 3))) & 1) != 0)) ? sc[t][e] : NEG_INF;
              }
          }
          if (fresh) {
            const float mx = top();
            m_run = m_run == NEG_INF ? mx - kLift : m_run;
            fresh = __ballot(m_run == NEG_INF) != 0;
          }
        }
        // P^T = 2^(s + log2 s_v + kLift - m), so that s_v is in the exponent, and the sum takes it back
        float2 kv = scale[NG - 1], kv_next;
        float eg = 0.0f, sum = 0.0f, most = 0.0f, l_new = l_run;
        // The granules' order is NG - 1, 0, 1, ...: those of the tile before are used up in
        // the order 0, 1, ..., so that all but the first of the new ones take their place.
        u4v p_last;
        auto weigh = [&](int n) __attribute__((always_inline)) {  // two weights
          const int g = ((n >> 2) + NG - 1) % NG, e = 2 * (n & 3);
          if (e == 0) {
            if (n > 0) kv = kv_next;
            eg = kv.y - (m_run == NEG_INF ? 0.0f : m_run);
            sum = 0.0f;
          }
          if (e == 2 && n < 4 * NG - 4) kv_next = scale[(g + 1) % NG];
          const float u = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[g >> 1][8 * (g & 1) + e], kv.x, eg));
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[g >> 1][8 * (g & 1) + e + 1], kv.x, eg));
          (g == NG - 1 ? p_last : p[g])[n & 3] = F::pack(u, w);
          sum += u;
          sum += w;
          if (e == 6) {  // the sum of the probabilities takes s_v back
            l_new = __builtin_fmaf(sum, __builtin_amdgcn_exp2f(-kv.y), l_new);
            most = __builtin_fmaxf(most, sum);
          }
        };

        constexpr int NP = 4 * NG, AHEAD = 2;  // pairs of weights; slices a fragment is read ahead
        const uint8_t* kt = sK[buf ^ 1];
        const uint8_t* vt = sK[2 + (buf ^ 1)];
        u4v kf[AHEAD + 1], vf[AHEAD + 1], qf[2];
        qf[0] = q_frag(0);
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) {
          kf[n] = k_frag(kt, n);
          vf[n] = v_frag(vt, n / DT, n % DT);
        }
#pragma unroll
        for (int t = 0; t < NH; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) sn[t][e] = 0.0f;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          if (n + AHEAD < NS) {
            kf[(n + AHEAD) % (AHEAD + 1)] = k_frag(kt, n + AHEAD);
            vf[(n + AHEAD) % (AHEAD + 1)] = v_frag(vt, (n + AHEAD) / DT, (n + AHEAD) % DT);
          }
          if (n % NH == 0 && n + NH < NS) qf[(n / NH + 1) & 1] = q_frag(n / NH + 1);
          sn[n % NH] = O::mfma(kf[n % (AHEAD + 1)], qf[(n / NH) & 1], sn[n % NH]);
#pragma unroll
          for (int w = n * NP / NS; w < (2 * n + 1) * NP / (2 * NS); ++w) weigh(w);
          acc[n % DT] = F::mfma(vf[n % (AHEAD + 1)], p[n / DT], acc[n % DT]);
#pragma unroll
          for (int w = (2 * n + 1) * NP / (2 * NS); w < (n + 1) * NP / NS; ++w) weigh(w);
          // (one piece of the next codes into LDS every few slices, then the loads)
#pragma unroll
          for (int c = 0; c < PIECES; ++c)
            if (n == (c + 1) * NS / (PIECES + 2)) store_piece(c, buf, raw[c]);
          if (n == (PIECES + 1) * NS / (PIECES + 2))
            load_codes(i + 3, (i & (TB - 1)) >= TB - 3 ? ahead.page : now.page, i + 1, (i & (TB - 1)) == TB - 1 ? ahead.page : now.page, raw);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (__builtin_expect(__ballot(most > 60000.0f) != 0, 0)) {
#pragma unroll
          for (int t = 0; t < NH; ++t) asm volatile("" : "+v"(sc[t]));  // (nothing of this is to be done before the branch)
          const float nx = __builtin_fmaxf(m_run, top() - kLift);
          const float alpha = nx == m_run ? 1.0f : __builtin_amdgcn_exp2f(m_run - nx);
          m_run = nx;
          l_new = l_run * alpha;
          kv = scale[NG - 1];
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[d][e] *= alpha;
#pragma unroll
          for (int n = 0; n < NP; ++n) weigh(n);
        }
        l_run = l_new;
        p[NG - 1] = p_last;
        if (__builtin_expect(i > 0 && partial(tile_at(i - 1)), 0)) put_nan(tile_at(i - 1), buf ^ 1);
        lds_barrier();
      };

      lds_barrier();  // the last segment's reads, and sNan
      {
        now = load_pages(0);
        ahead = load_pages(1);
        load_scales(0, now);
        uint4 first[PIECES];
        load_codes(0, now.page, 0, now.page, first);
        load_codes(1, now.page, 0, now.page, raw);
        if constexpr (QL) {
#pragma unroll
          for (int k = 0; k < KS; ++k) sQ[wave][k][lane] = q[k];  // (read by the lane that wrote it)
        }
        use(0, now);
        // (V's buffer of the tile before the first: zeros)
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
          if (!is_v(c)) store_piece(c, 0, first[c]);
          store_piece(c, 1, is_v(c) ? make_uint4(0, 0, 0, 0) : raw[c]);
        }
        load_codes(2, now.page, 0, now.page, raw);
#pragma unroll
        for (int g = 0; g < NG; ++g) p[g] = u4v{0, 0, 0, 0};
      }
      lds_barrier();
      v16f s0[NH], s1[NH];
#pragma unroll
      for (int t = 0; t < NH; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) s0[t][e] = 0.0f;
#pragma unroll
      for (int n = 0; n < NS; ++n) s0[n % NH] = O::mfma(k_frag(sK[0], n), q_frag(n / NH), s0[n % NH]);
      lds_barrier();
      for (int i = 0; i < n_tiles; i += 2) {
        tile_step(i, 0, s0, s1);
        if (i + 1 >= n_tiles) break;
        tile_step(i + 1, 1, s1, s0);
      }
      const int lb = (n_tiles - 1) & 1;
#pragma unroll
      for (int n = 0; n < NS; ++n)
        acc[n % DT] = F::mfma(v_frag(sK[2] + lb * kKeys * ROW, n / DT, n % DT), p[n / DT], acc[n % DT]);
      put_nan(tile_at(n_tiles - 1), lb);
    }

    // ---- out
    l_run += __shfl_xor(l_run, 32, 64);
    if (live) {
      const int64_t at = (int64_t)(s.row0 + tq) * (a.Hkv * a.G) + hq;
      if (whole && !(MODE == kShared && a.raw)) {
        Kv8Join join = kv8_join<MODE>(a, s, at, hq, m_run, l_run);
        join.own *= kUnlift;
        uint16_t* o = a.o + at * a.D + 4 * g2;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (32 * d + 8 * k < a.D) {
              const float4 y = kv8_joined<MODE>(a, join, at, 32 * d + 8 * k + 4 * g2,
                                          make_float4(acc[d][4 * k], acc[d][4 * k + 1], acc[d][4 * k + 2], acc[d][4 * k + 3]));
              *reinterpret_cast<uint2*>(o + 32 * d + 8 * k) = make_uint2(kv8_out2<QT>(y.x, y.y), kv8_out2<QT>(y.z, y.w));
            }
      } else {
        float* o = (MODE == kShared && whole ? a.prior_acc + at * a.D : a.ws_acc + (slot * RT + r) * a.D) + 4 * g2;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (32 * d + 8 * k < a.D)
              *reinterpret_cast<float4*>(o + 32 * d + 8 * k) =
                  make_float4(acc[d][4 * k] * kUnlift, acc[d][4 * k + 1] * kUnlift, acc[d][4 * k + 2] * kUnlift,
                              acc[d][4 * k + 3] * kUnlift);
        if (g2 == 0)
          *reinterpret_cast<float2*>(MODE == kShared && whole ? a.prior_ml + 2 * at : a.ws_ml + (slot * RT + r) * 2) = make_float2(m_run, l_run);
      }
    }
  }
}

template <int DP, int QT, int MODE>
void launch_prefill(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t st) {
  constexpr int NW = DP == 128 ? 8 : 4, RT = 32 * NW;
  static_assert(RT == kv8_chunk_rows(DP), "the plan's row tile");
  const int64_t items = p.items;
  if (p.parts == 0) {
    kv8_prefill_kernel<DP, QT, NW, false, MODE><<<(unsigned)items, 64 * NW, 0, st>>>(a, items);
  } else {
    kv8_prefill_kernel<DP, QT, NW, true, MODE><<<a.parts * a.Hkv, 64 * NW, 0, st>>>(a, items);
    kv8_merge_kernel<RT, chunk_keys(DP), QT, MODE><<<(unsigned)(items * (RT / 4)), 256, 0, st>>>(a);
  }
}

template <int QT, int MODE>
void launch_prefill_as(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t st) {
  if (a.D <= 64)
    launch_prefill<64, QT, MODE>(a, p, st);
  else if (a.D <= 128)
    launch_prefill<128, QT, MODE>(a, p, st);
  else
    launch_prefill<256, QT, MODE>(a, p, st);
}

template <int QT>
void launch_mode(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t st) {
  if (kv8_mode(a) == kPlain)
    launch_prefill_as<QT, kPlain>(a, p, st);
  else if (kv8_mode(a) == kFirst)
    launch_prefill_as<QT, kFirst>(a, p, st);
  else
    launch_prefill_as<QT, kShared>(a, p, st);
}

}  // namespace

void launch_kv8_prefill(const Kv8AttnArgs& a, const Kv8AttnPlan& p, int dtype, hipStream_t st) {
  if (dtype == SGL_BF16)
    launch_mode<SGL_BF16>(a, p, st);
  else
    launch_mode<SGL_F16>(a, p, st);
}

}  // namespace sgl
