// Attention over the 8-bit paged cache: few rows a sequence and head (decode,
// draft tokens, short chunks).
//
//   s_j = (q . code_j) s_k[block j] scale,  o = sum_j 2^(s_j - m) code_j s_v[block j] / sum_j 2^(s_j - m)
// over the keys j that the row sees, in one pass with a running reference m.
//
// Bound by HBM: a key and its value are D bytes each and read once (128 sequences up
// to 16384 keys, 4 heads of 128: 186 us with the merge, 6.2 TB/s in the kernel).  So the
// codes go straight from memory into the registers of the lanes that need
// them, 32 tokens a wavefront and step, the next step's in flight; no LDS and no
// barrier until an item ends.  Both products are v_mfma_f32_16x16x32:
//   S^T = K . Q^T: lane (row m = lane % 16, g = lane / 16) takes token m of a
//     granule of 16 and 16-byte pieces 4 i + g of its row (the order of the
//     contraction is free as long as q follows it);
//   O^T = V^T . P^T: the output layout of S^T is the B operand layout of P^T
//     when slot j of k-group g stands for token 4 g + j of the first granule
//     (j < 4) or 4 g + j - 4 of the second.  Lane (m, g) loads those 8 tokens'
//     C = D / 16 bytes from C m on, transposes them in registers (v_perm), and
//     holds the A operands of C tiles of 16 dims (row m of tile j: dim C m + j).
// A conversion e4m3 -> bf16 (exact) is one instruction for two codes.  The
// scales are one number for 16 tokens: s_k multiplies the score, log2 s_v is added
// to it, so that P carries s_v.  P and the codes of V are f16 for every type of q: a
// code is exact there, a weight is rounded by at most 2^-11 of itself (bf16: 2^-8) or
// 2^-35 of the row's largest (kLift), and that is the only rounding between the codes
// and the output's own.
#include "sgl_kv8_attn.h"

namespace sgl {
namespace {

typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kTile = 32 * kWaves;  // tokens of a key tile: one step of every wavefront

template <int QT>
struct Op;
template <>
struct Op<SGL_BF16> {
  typedef v8bf V;
  static __device__ __forceinline__ v4f mfma(V a, V b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ __forceinline__ uint32_t cvt(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  }
};
template <>
struct Op<SGL_F16> {
  typedef v8h V;
  static __device__ __forceinline__ v4f mfma(V a, V b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ __forceinline__ uint32_t cvt(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
  }
};

// 8 codes -> 8 values of the product's type
template <int QT>
__device__ __forceinline__ typename Op<QT>::V cvt8(uint32_t lo, uint32_t hi) {
  const u4v w = {Op<QT>::template cvt<false>(lo), Op<QT>::template cvt<true>(lo), Op<QT>::template cvt<false>(hi),
                Op<QT>::template cvt<true>(hi)};
  return __builtin_bit_cast(typename Op<QT>::V, w);
}

// byte k of a, b, c, d as word k
__device__ __forceinline__ void transpose4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t* o) {
  const uint32_t ab0 = __builtin_amdgcn_perm(b, a, 0x05010400u), ab1 = __builtin_amdgcn_perm(b, a, 0x07030602u);
  const uint32_t cd0 = __builtin_amdgcn_perm(d, c, 0x05010400u), cd1 = __builtin_amdgcn_perm(d, c, 0x07030602u);
  o[0] = __builtin_amdgcn_perm(cd0, ab0, 0x05040100u);
  o[1] = __builtin_amdgcn_perm(cd0, ab0, 0x07060302u);
  o[2] = __builtin_amdgcn_perm(cd1, ab1, 0x05040100u);
  o[3] = __builtin_amdgcn_perm(cd1, ab1, 0x07060302u);
}

// The codes of one step: 32 tokens.
template <int DP>
struct Codes {
  uint4 k[2][DP / 64];
  uint32_t v[8][DP / 64];  // tokens as above, C = DP / 16 bytes each
};

// Codes that one workgroup reads, or several (which the nontemporal policy would have all
// read from memory).
template <class V, bool ONCE>
__device__ __forceinline__ V ld_codes(const uint8_t* p) {
  if constexpr (!ONCE)
    return *reinterpret_cast<const V*>(p);
  else if constexpr (sizeof(V) == 16)
    return ld16_stream(p);
  else
    return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
}

// What the wavefronts of a workgroup join their sums through, a column tile at a time.
template <int DP>
struct Joint {
  __align__(16) float acc[kWaves][16][DP + 4];
  float m[kWaves][16], l[kWaves][16];
};

// One segment.  DP: head dim rounded up to 64, 128 or 256; NC: 16-row column tiles
template <int DP, int NC, int QT, int MODE, bool ONCE = true>
__device__ __forceinline__ void few_segment(const Kv8AttnArgs& a, const Kv8Segment& seg, int head, Joint<DP>& lds) {
  constexpr int RT = 16 * NC, KI = DP / 64, C = DP / 16, W = C / 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, g = lane >> 4;
  const float NEG_INF = -__builtin_huge_valf();
  {
    const Kv8Seq& s = seg.s;
    const int b = seg.b, rt = seg.rt, t0 = seg.t0, t1 = seg.t1;
    const int rows = s.n * a.G - rt * RT;  // valid rows of the tile (may be more than RT)
    const bool causal = a.causal && !(MODE == kJoint && s.group == kIsGroup);

    // the rows: their queries and what they see
    typename Op<QT>::V q[NC][2 * KI];
    int hi[NC], lo[NC];
    int all_hi = s.len, all_lo = 0;  // what every row of the tile sees
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int r = 16 * c + m;
      const bool live = r < rows;
      const int row = rt * RT + (live ? r : 0), t = row / a.G, h = head * a.G + (row - t * a.G);
      const int pos = s.len - s.n + t;
      hi[c] = !live ? 0 : causal ? pos + 1 : s.len;
      lo[c] = causal && a.window > 0 ? pos - a.window + 1 : 0;
      const uint16_t* src = a.q + (int64_t)(s.row0 + t) * a.qt + (int64_t)h * a.qh;
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int d = 64 * i + 16 * g;
        uint4 u = make_uint4(0, 0, 0, 0), w = u;
        if (live && d < a.D) {
          u = *reinterpret_cast<const uint4*>(src + d);
          w = *reinterpret_cast<const uint4*>(src + d + 8);
        }
        q[c][2 * i] = __builtin_bit_cast(typename Op<QT>::V, u);
        q[c][2 * i + 1] = __builtin_bit_cast(typename Op<QT>::V, w);
      }
    }
    if (causal) {
      const int last = rows < RT ? rows - 1 : RT - 1;
      const int p0 = s.len - s.n + (rt * RT) / a.G, p1 = s.len - s.n + (rt * RT + last) / a.G;
      all_hi = p0 + 1 < all_hi ? p0 + 1 : all_hi;
      if (a.window > 0) all_lo = p1 - a.window + 1;
    }

    v4f acc[NC][C];
    float m_run[NC], l_run[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      m_run[c] = NEG_INF;
      l_run[c] = 0.0f;
#pragma unroll
      for (int j = 0; j < C; ++j) acc[c][j] = v4f{0, 0, 0, 0};
    }

    const int32_t* table = a.pages + (int64_t)(MODE == kJoint ? s.table_row : MODE == kShared && a.table_row ? a.table_row[b] : b) * a.row_pages;
    const int pmask = (1 << a.page_shift) - 1;
    // the wavefront's first token in step i; only the last tile's may lie behind the end
    auto token = [&](int i) __attribute__((always_inline)) { return s.template tile<MODE>(t0 + i) * kTile + 32 * wave; };
    const int steps = t1 - t0 - (token(t1 - t0 - 1) < s.len ? 0 : 1);

    // Pages and scales of 32 steps at a time: lane l has granule l & 1 of step l >> 1.
    // Loaded a batch ahead, so that no step waits for its table entry.
    struct Batch {
      int page;  // 0 where there is none
      float ks, vs;
      bool ok;
    };
    auto load_pages = [&](int batch) __attribute__((always_inline)) {
      Batch o;
      const int t = token(32 * batch + (lane >> 1)) + 16 * (lane & 1);
      const int page = table[(t < s.len ? t : s.len - 1) >> a.page_shift];
      o.ok = t < s.len && page >= 0 && page < a.n_pages;
      o.page = o.ok ? page : 0;
      return o;
    };
    auto load_scales = [&](int batch, Batch& o) __attribute__((always_inline)) {
      const int t = token(32 * batch + (lane >> 1)) + 16 * (lane & 1);
      const int64_t piece = (((int64_t)o.page * a.Hkv + head) << (a.page_shift - a.block_shift)) +
                            ((t & pmask) >> a.block_shift);
      o.ks = a.ks[piece];
      o.vs = a.vs[piece];
    };

    // lane offsets; dims behind D repeat others of the same token, whose scores
    // meet zeros of q and whose outputs are not stored
    int kd[KI], vd;
#pragma unroll
    for (int i = 0; i < KI; ++i) kd[i] = m * a.D + (64 * i + 16 * g < a.D ? 64 * i + 16 * g : 0);
    vd = 4 * g * a.D + (C * m < a.D ? C * m : 0);
    auto load = [&](int i, int pages, Codes<DP>& r) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int page = __builtin_amdgcn_readlane(pages, 2 * (i & 31) + u);
        const int spot = (token(i) + 16 * u) & pmask;
        const int64_t row = ((((int64_t)page * a.Hkv + head) << a.page_shift) + spot) * a.D;
        const uint8_t* kp = a.kc + row;
        const uint8_t* vp = a.vc + row;
#pragma unroll
        for (int k = 0; k < KI; ++k) r.k[u][k] = ld_codes<uint4, ONCE>(kp + (uint32_t)kd[k]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint8_t* at = vp + j * a.D + (uint32_t)vd;
          if constexpr (W == 1) {
            r.v[4 * u + j][0] = ld_codes<uint32_t, ONCE>(at);
          } else if constexpr (W == 2) {
            const u2v y = ld_codes<u2v, ONCE>(at);
            r.v[4 * u + j][0] = y.x;
            r.v[4 * u + j][1] = y.y;
          } else {
            const uint4 y = ld_codes<uint4, ONCE>(at);
            r.v[4 * u + j][0] = y.x;
            r.v[4 * u + j][1] = y.y;
            r.v[4 * u + j][2] = y.z;
            r.v[4 * u + j][3] = y.w;
          }
        }
      }
    };

    // acc += V^T . P^T for the codes v of the step
    auto accumulate = [&](const uint32_t (*v)[W], const v8h* p) __attribute__((always_inline)) {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        uint32_t x0[4], x1[4];
        transpose4(v[0][w], v[1][w], v[2][w], v[3][w], x0);
        transpose4(v[4][w], v[5][w], v[6][w], v[7][w], x1);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const v8h f = cvt8<SGL_F16>(x0[k], x1[k]);
#pragma unroll
          for (int c = 0; c < NC; ++c) acc[c][4 * w + k] = Op<SGL_F16>::mfma(f, p[c], acc[c][4 * w + k]);
        }
      }
    };

    float kcs, evs, ivs;  // of the batch: score scale, kLift + log2 of the value scale, 2^-that
    uint64_t okm;  // granules that are there, with scales as they should be
    auto use = [&](const Batch& o) __attribute__((always_inline)) {
      // (what was never written may hold anything)
      const bool good = kv8_scale_ok(o.ks) && kv8_scale_ok(o.vs);
      kcs = !o.ok ? 0.0f : good ? o.ks * a.c1 : __builtin_nanf("");
      evs = kv8_exponent(o.ok, good, o.vs);
      ivs = __builtin_amdgcn_exp2f(-evs);
      okm = __ballot(evs < kNoToken && evs != kNoValue);
    };
    auto lane_f = [&](float v, int l) { return bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(v), l)); };

    auto step = [&](int at, Codes<DP>& r) __attribute__((always_inline)) {
      const int tok = token(at), l0 = 2 * (at & 31);
      const uint32_t ok = (uint32_t)(okm >> l0) & 3u;
      v4f sc[NC][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int c = 0; c < NC; ++c) sc[c][u] = v4f{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < KI; ++i) {
          const typename Op<QT>::V k0 = cvt8<QT>(r.k[u][i].x, r.k[u][i].y), k1 = cvt8<QT>(r.k[u][i].z, r.k[u][i].w);
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            sc[c][u] = Op<QT>::mfma(k0, q[c][2 * i], sc[c][u]);
            sc[c][u] = Op<QT>::mfma(k1, q[c][2 * i + 1], sc[c][u]);
          }
        }
      }
      const bool plain = tok + 32 <= all_hi && (tok >= all_lo || (MODE == kFirst && tok + 32 <= a.first)) && ok == 3;
      const uint32_t here = plain ? 3u : (uint32_t)(__ballot(evs != kNoToken) >> l0) & 3u;
      uint32_t seen[NC];  // bit 4 u + i: the row sees token 16 u + 4 g + i
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        seen[c] = 0xFF;
        if (!plain) {
          seen[c] = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = tok + 16 * (i >> 2) + 4 * g + (i & 3);
            const bool in = MODE == kFirst ? (uint32_t)(key - a.first) >= (uint32_t)(lo[c] > a.first ? lo[c] - a.first : 0) : key >= lo[c];
            if (key < hi[c] && in && key < s.len && ((here >> (i >> 2)) & 1u)) seen[c] |= 1u << i;
          }
        }
      }
      // P^T = 2^(s + log2 s_v + kLift - m): the value's scale is part of the exponent, so
      // that P fits f16 as well, and the sum of the probabilities takes both back
      float kc[2], ev[2], iv[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        kc[u] = lane_f(kcs, l0 + u);
        ev[u] = lane_f(evs, l0 + u);
        iv[u] = lane_f(ivs, l0 + u);
      }
      v8h p[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __builtin_fmaf(sc[c][i >> 2][i & 3], kc[i >> 2], ev[i >> 2]);
        if (!plain) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = (seen[c] >> i) & 1u ? f[i] : NEG_INF;
        }
        float mx = f[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = __builtin_fmaxf(mx, f[i]);
        // The reference moves only when a weight's exponent exceeds it by more than 15.5
        // (log2 units), to kLift below: any reference gives the same softmax, the
        // weights fit f16, and the accumulators are rarely rescaled.
        if (__ballot(!(mx <= m_run[c] + 15.5f) && mx != NEG_INF)) {
          mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16, 64));
          mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32, 64));
          const float next = mx <= m_run[c] + 15.5f ? m_run[c] : __builtin_fmaxf(m_run[c], mx - kLift);
          const float alpha = next == m_run[c] ? 1.0f : __builtin_amdgcn_exp2f(m_run[c] - next);
          m_run[c] = next;
          l_run[c] *= alpha;
#pragma unroll
          for (int j = 0; j < C; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[c][j][i] *= alpha;
        }
        const float ref = m_run[c] == NEG_INF ? 0.0f : m_run[c];
        float l = 0.0f;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          f[i] = __builtin_amdgcn_exp2f(f[i] - ref);
          l = __builtin_fmaf(f[i], iv[i >> 2], l);
        }
        l_run[c] += l;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack2<SGL_F16>(f[2 * i], f[2 * i + 1]);
        p[c] = __builtin_bit_cast(v8h, u4v{w[0], w[1], w[2], w[3]});
      }
      if (!plain) {
        // What no row sees must not reach the product: keys behind the last
        // (never written) are zeroed.  A NaN code that some rows see and others
        // do not is zeroed too and put back into the sums of those that do.
        const uint32_t none = (uint32_t)(__ballot(evs == kNoValue) >> l0) & 3u;
        uint32_t nan[8][W], any = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool there = tok + 16 * (j >> 2) + 4 * g + (j & 3) < s.len && ((here >> (j >> 2)) & 1u);
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const uint32_t v = there ? r.v[j][w] : 0u;
            const uint32_t bad = (((v & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;
            any |= bad;
            nan[j][w] = bad * 0x38u;  // 1.0
            r.v[j][w] = (none >> (j >> 2)) & 1u ? 0u : v & ~(bad * 0xFFu);
          }
        }
        if (__ballot(any != 0)) {
#pragma unroll
          for (int w = 0; w < W; ++w) {
            uint32_t x0[4], x1[4];
            transpose4(nan[0][w], nan[1][w], nan[2][w], nan[3][w], x0);
            transpose4(nan[4][w], nan[5][w], nan[6][w], nan[7][w], x1);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const v8bf f = cvt8<SGL_BF16>(x0[k], x1[k]);
#pragma unroll
              for (int c = 0; c < NC; ++c) {
                u4v e;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  e[i] = ((seen[c] >> (2 * i)) & 1u) * 0x3F80u | ((seen[c] >> (2 * i + 1)) & 1u) * 0x3F800000u;
                const v4f hit = Op<SGL_BF16>::mfma(f, __builtin_bit_cast(v8bf, e), v4f{0, 0, 0, 0});
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (hit[i] > 0.0f) acc[c][4 * w + k][i] = __builtin_nanf("");
              }
            }
          }
        }
      }
      accumulate(r.v, p);
    };

    if (steps > 0) {
      // The next step's codes are on their way while one is worked on (two steps ahead
      // is no faster: 128 sequences up to 16384 keys 190 us against 186).
      // Loads are never under a branch (behind the last step they repeat it), so that
      // the waits count them instead of draining them.
      Batch now = load_pages(0), ahead = load_pages(1);
      load_scales(0, now);
      Codes<DP> r0, r1;
      load(0, now.page, r0);
      use(now);
      for (int i = 0; i < steps; i += 2) {
        if ((i & 31) == 0 && i > 0) {
          now = ahead;
          use(now);
          ahead = load_pages((i >> 5) + 1);
        }
        if ((i & 31) == 16) load_scales((i >> 5) + 1, ahead);
        load(i + 1 < steps ? i + 1 : i, now.page, r1);
        step(i, r0);
        if (i + 1 >= steps) break;
        const int n = i + 2 < steps ? i + 2 : i + 1;
        load(n, (n & 31) == 0 ? ahead.page : now.page, r0);
        step(i + 1, r1);
      }
    }

    // join the wavefronts, a column tile at a time
    const bool whole = t0 == 0 && t1 == s.tiles;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (t0 == 0 ? 1 : 0);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float l = l_run[c];
      l += __shfl_xor(l, 16, 64);
      l += __shfl_xor(l, 32, 64);
      __syncthreads();
      if (g == 0) {
        lds.m[wave][m] = m_run[c];
        lds.l[wave][m] = l;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < C; j += 4)
          *reinterpret_cast<float4*>(&lds.acc[wave][m][C * (4 * g + i) + j]) =
              make_float4(acc[c][j][i], acc[c][j + 1][i], acc[c][j + 2][i], acc[c][j + 3][i]);
      __syncthreads();
      const int chunks = a.D >> 3;
      for (int i = threadIdx.x; i < 16 * chunks; i += 64 * kWaves) {
        const int n = i / chunks, d = (i - n * chunks) << 3, r = 16 * c + n;
        if (r >= rows) break;
        float M = NEG_INF;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = __builtin_fmaxf(M, lds.m[w][n]);
        const float ref = M == NEG_INF ? 0.0f : M;
        float sum = 0.0f, y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float f = __builtin_amdgcn_exp2f(lds.m[w][n] - ref);
          sum += lds.l[w][n] * f;
#pragma unroll
          for (int v = 0; v < 8; ++v) y[v] += lds.acc[w][n][d + v] * (f * kUnlift);
        }
        if (whole) {
          const int row = rt * RT + r, t = row / a.G, h = head * a.G + (row - t * a.G);
          const int64_t at = (int64_t)(s.row0 + t) * (a.Hkv * a.G) + h;
          float4 y0 = make_float4(y[0], y[1], y[2], y[3]), y1 = make_float4(y[4], y[5], y[6], y[7]);
          if (MODE == kJoint || (MODE == kShared && a.raw)) {
            const bool prior = MODE == kShared || s.group == kIsGroup;
            float4* out = reinterpret_cast<float4*>((prior ? a.prior_acc : a.own_acc) + at * a.D + d);
            out[0] = y0;
            out[1] = y1;
            if (d == 0) *reinterpret_cast<float2*>((prior ? a.prior_ml : a.own_ml) + 2 * at) = make_float2(M, sum);
          } else {
            const Kv8Join join = kv8_join<MODE>(a, s, at, h, M, sum);
            y0 = kv8_joined<MODE>(a, join, at, d, y0);
            y1 = kv8_joined<MODE>(a, join, at, d + 4, y1);
            *reinterpret_cast<uint4*>(a.o + at * a.D + d) =
                make_uint4(kv8_out2<QT>(y0.x, y0.y), kv8_out2<QT>(y0.z, y0.w), kv8_out2<QT>(y1.x, y1.y),
                           kv8_out2<QT>(y1.z, y1.w));
          }
        } else {
          float4* out = reinterpret_cast<float4*>(a.ws_acc + (slot * (MODE == kJoint ? a.slot_rows : RT) + r) * a.D + d);
          out[0] = make_float4(y[0], y[1], y[2], y[3]);
          out[1] = make_float4(y[4], y[5], y[6], y[7]);
          if (d == 0) *reinterpret_cast<float2*>(a.ws_ml + (slot * (MODE == kJoint ? a.slot_rows : RT) + r) * 2) = make_float2(M, sum);
        }
      }
    }
  }
}

// SPLIT: workgroups share the lines, else a workgroup takes a whole item
template <int DP, int NC, int QT, bool SPLIT, int MODE>
__global__ __launch_bounds__(64 * kWaves, DP == 64 ? 2 : 1) void kv8_attn_few_kernel(const Kv8AttnArgs a) {
  __shared__ Joint<DP> lds;
  constexpr int RT = 16 * NC;
  int head, part = 0;
  Kv8Segment seg;
  if constexpr (SPLIT) {
    Kv8Walk<RT, kTile, MODE> walk;
    kv8_wg_at(a, (int)blockIdx.x, &head, &part);
    if (!walk.start(a, part)) return;
    while (walk.next(a, seg)) few_segment<DP, NC, QT, MODE>(a, seg, head, lds);
  } else {
    if (kv8_item<RT, kTile, MODE>(a, (int64_t)blockIdx.x, &head, seg)) few_segment<DP, NC, QT, MODE>(a, seg, head, lds);
  }
}

// Sequences and groups on one line, in tiles of NC and NCG column tiles.
// WGS workgroups a CU.
template <int DP, int NCG, int NC, int QT, int WGS>
__global__ __launch_bounds__(64 * kWaves, WGS) void kv8_joint_kernel(const Kv8AttnArgs a) {
  __shared__ Joint<DP> lds;
  int head, part = 0;
  Kv8Segment seg;
  Kv8Walk<16 * NC, kTile, kJoint> walk;
  kv8_wg_at(a, (int)blockIdx.x, &head, &part);
  if (!walk.start(a, part)) return;
  while (walk.next(a, seg)) {
    if (seg.s.group == kIsGroup)
      few_segment<DP, NCG, QT, kJoint, false>(a, seg, head, lds);
    else
      few_segment<DP, NC, QT, kJoint>(a, seg, head, lds);
  }
}

template <int DP, int NC, int QT, int MODE>
void launch_few_as(const Kv8AttnArgs& a, int64_t items, hipStream_t st) {
  if (a.parts == 0) {
    kv8_attn_few_kernel<DP, NC, QT, false, MODE><<<(unsigned)items, 64 * kWaves, 0, st>>>(a);
    return;
  }
  kv8_attn_few_kernel<DP, NC, QT, true, MODE><<<a.parts * a.Hkv, 64 * kWaves, 0, st>>>(a);
  kv8_merge_kernel<16 * NC, kTile, QT, MODE><<<(unsigned)(items * 4 * NC), 256, 0, st>>>(a);
}

template <int DP, int NC, int QT>
void launch_few(const Kv8AttnArgs& a, int64_t items, hipStream_t st) {
  if (kv8_mode(a) == kPlain)
    launch_few_as<DP, NC, QT, kPlain>(a, items, st);
  else if (kv8_mode(a) == kFirst)
    launch_few_as<DP, NC, QT, kFirst>(a, items, st);
  else
    launch_few_as<DP, NC, QT, kShared>(a, items, st);
}

template <int QT>
void launch_attn(Kv8AttnArgs a, const Kv8AttnPlan& p, hipStream_t st) {
  a.parts = (int)p.parts;
  a.above = (int)p.above;
  a.upto = (int)p.upto;
  a.ws_ml = a.ws_acc + 2 * p.parts * a.Hkv * p.row_tile * a.D;
  if (p.row_tile > 32)
    launch_kv8_prefill(a, p, QT, st);
  else if (a.D <= 64)
    p.row_tile == 16 ? launch_few<64, 1, QT>(a, p.items, st) : launch_few<64, 2, QT>(a, p.items, st);
  else if (a.D <= 128)
    p.row_tile == 16 ? launch_few<128, 1, QT>(a, p.items, st) : launch_few<128, 2, QT>(a, p.items, st);
  else
    launch_few<256, 1, QT>(a, p.items, st);
}

template <int DP, int NCG, int NC, int QT>
void launch_joint_as(const Kv8AttnArgs& a, const Kv8JointPlan& p, hipStream_t st) {
  const dim3 grid(a.parts * a.Hkv), threads(64 * kWaves);
  // (what the plan says of these heads and tiles: always two, either, always one)
  if constexpr (DP == 64) {
    kv8_joint_kernel<DP, NCG, NC, QT, 2><<<grid, threads, 0, st>>>(a);
  } else if constexpr (DP == 128 && NCG == 2) {
    if (p.per_cu == 2)
      kv8_joint_kernel<DP, NCG, NC, QT, 2><<<grid, threads, 0, st>>>(a);
    else
      kv8_joint_kernel<DP, NCG, NC, QT, 1><<<grid, threads, 0, st>>>(a);
  } else {
    kv8_joint_kernel<DP, NCG, NC, QT, 1><<<grid, threads, 0, st>>>(a);
  }
  const int64_t rows = (int64_t)a.T * a.Hkv * a.G;
  kv8_joint_merge_kernel<16 * NC, kTile, QT><<<(unsigned)ceil_div(rows, 4), 256, 0, st>>>(a);
}
template <int DP, int QT>
void launch_joint_dim(const Kv8AttnArgs& a, const Kv8JointPlan& p, hipStream_t st) {
  if (p.group_rows == 16)
    launch_joint_as<DP, 1, 1, QT>(a, p, st);
  else if (p.row_tile == 16)
    launch_joint_as<DP, 2, 1, QT>(a, p, st);
  else if constexpr (DP <= 128)
    launch_joint_as<DP, 2, 2, QT>(a, p, st);
}
template <int QT>
void launch_joint(const Kv8AttnArgs& a, const Kv8JointPlan& p, hipStream_t st) {
  if (a.D <= 64)
    launch_joint_dim<64, QT>(a, p, st);
  else if (a.D <= 128)
    launch_joint_dim<128, QT>(a, p, st);
  else
    launch_joint_dim<256, QT>(a, p, st);
}

struct AttnPlans {
  Kv8AttnPlan p[2];  // one launch, or (chunks and few rows in one batch) two, one after the other on the same workspace
};
AttnPlans attn_plans(int64_t T, int64_t B, int Hkv, int G, int D, int64_t tokens, bool window = false) {
  const int cus = device_cu_count();
  return {{kv8_attn_plan(T, B, Hkv, G, D, tokens, cus, window), kv8_attn_rest(T, B, Hkv, G, D, tokens, cus, window)}};
}
size_t attn_workspace(const AttnPlans& plans, int Hkv, int D) {
  const size_t x = kv8_attn_workspace(plans.p[0], Hkv, D), y = kv8_attn_workspace(plans.p[1], Hkv, D);
  return x > y ? x : y;
}
bool attn_sizes_ok(int64_t T, int64_t B, int Hkv, int G, int D, int64_t max_tokens) {
  return T >= 0 && B >= 0 && Hkv >= 1 && G >= 1 && D >= 16 && max_tokens >= 0;
}

// Checks a call's arguments and lays them out; `nothing`: there is no row to write.
struct AttnCall {
  const void* q;
  int64_t q_token_stride, q_head_stride;
  int dtype;
  int64_t T, B;
  int Hkv, G, D;
  const int32_t *cu_tokens, *lens, *block_table;
  int64_t row_pages;
  int page_size, block;
  int64_t n_pages;
  const void *k_codes, *v_codes;
  const float *k_scale, *v_scale;
  float softmax_scale;
  int causal;
  int64_t window;
  const float* sink;
  void* out;
  void* workspace;
};
int attn_args(const AttnCall& c, Kv8AttnArgs& a, bool& nothing) {
  const int64_t T = c.T, B = c.B;
  SGL_REQUIRE(c.dtype == SGL_BF16 || c.dtype == SGL_F16, "kv8_attn: dtype %d (bf16 or f16)", c.dtype);
  const int rc = kv8_check_cache("kv8_attn", c.Hkv, c.D, c.page_size, c.block, c.n_pages, c.row_pages);
  if (rc != SGL_OK) return rc;
  SGL_REQUIRE(c.G >= 1 && (int64_t)c.G * c.Hkv <= 65536, "kv8_attn: G=%d query heads for each of %d kv heads", c.G, c.Hkv);
  SGL_REQUIRE(T >= 0 && B >= 0 && B <= (1 << 24) && T * c.G < (1ll << 31), "kv8_attn: T=%lld B=%lld out of range",
              (long long)T, (long long)B);
  SGL_REQUIRE(c.cu_tokens || T == B, "kv8_attn: without cu_tokens every sequence has one token (T=%lld, B=%lld)",
              (long long)T, (long long)B);
  SGL_REQUIRE(c.window >= 0 && (c.causal || c.window == 0), "kv8_attn: a window (%lld) is for causal attention",
              (long long)c.window);
  SGL_REQUIRE(c.softmax_scale > 0.0f && c.softmax_scale < 1e30f, "kv8_attn: softmax_scale must be positive");
  nothing = T == 0 || B == 0;
  if (nothing) return SGL_OK;
  SGL_REQUIRE(c.q && c.lens && c.block_table && c.k_codes && c.v_codes && c.k_scale && c.v_scale && c.out,
              "kv8_attn: null pointer");
  SGL_REQUIRE(aligned(c.q, 16) && c.q_token_stride % 8 == 0 && c.q_head_stride % 8 == 0,
              "kv8_attn: q and its strides must be 16-byte aligned");
  SGL_REQUIRE(aligned(c.k_codes, 16) && aligned(c.v_codes, 16) && aligned(c.out, 16),
              "kv8_attn: misaligned cache or output");
  const int64_t tokens = c.row_pages * c.page_size;
  a = Kv8AttnArgs{};
  a.q = (const uint16_t*)c.q;
  a.qt = c.q_token_stride;
  a.qh = c.q_head_stride;
  a.o = (uint16_t*)c.out;
  a.kc = (const uint8_t*)c.k_codes;
  a.vc = (const uint8_t*)c.v_codes;
  a.ks = c.k_scale;
  a.vs = c.v_scale;
  a.pages = c.block_table;
  a.lens = c.lens;
  a.cu = c.cu_tokens;
  a.sink = c.sink;
  a.n_pages = c.n_pages;
  a.T = (int)T;
  a.B = (int)B;
  a.Hkv = c.Hkv;
  a.G = c.G;
  a.D = c.D;
  a.row_pages = (int)c.row_pages;
  a.page_shift = __builtin_ctz((unsigned)c.page_size);
  a.block_shift = __builtin_ctz((unsigned)c.block);
  a.c1 = c.softmax_scale * kLog2e;
  a.window = c.window >= tokens ? 0 : (int)c.window;  // (as long as the table: all keys)
  a.causal = c.causal != 0;
  a.ws_acc = (float*)c.workspace;
  return SGL_OK;
}

int check_workspace(const void* workspace, size_t bytes, size_t need) {
  if (need && (!workspace || bytes < need)) {
    set_error("kv8_attn: workspace of %zu bytes, needs %zu", workspace ? bytes : 0, need);
    return SGL_ERR_WORKSPACE;
  }
  SGL_REQUIRE(aligned(workspace, 16), "kv8_attn: workspace must be 16-byte aligned");
  return SGL_OK;
}
int check_plans(const AttnPlans& plans, int64_t tokens) {
  for (const Kv8AttnPlan& p : plans.p)
    SGL_REQUIRE_SUPPORTED(p.items * ((tokens + 31) / 32 + kItemCost) < (1ll << 31) &&
                              p.items * p.row_tile / 4 < (1ll << 31),
                          "kv8_attn: %lld row tiles over %lld tokens are too many for one call", (long long)p.items,
                          (long long)tokens);
  return SGL_OK;
}
void launch_plans(const Kv8AttnArgs& a, int dtype, const AttnPlans& plans, hipStream_t st) {
  for (const Kv8AttnPlan& p : plans.p) {
    if (p.items == 0) continue;
    if (dtype == SGL_BF16)
      launch_attn<SGL_BF16>(a, p, st);
    else
      launch_attn<SGL_F16>(a, p, st);
  }
}

// ---- a common prefix: what its groups cover.
struct PrefixPlan {
  int32_t *cu, *lens, *row;  // of the groups: first token rows [n + 1], covered tokens, a row of the block table
  int32_t* skip;             // of the sequences: covered tokens
  Kv8Entry* entries;         // in their place, for one pass: of the sequences and behind them the groups
};
// Workgroup g takes group g; the last one the sequences of no group.
__global__ __launch_bounds__(256) void kv8_prefix_kernel(const Kv8AttnArgs a, const int32_t* cu_groups,
                                                         const int32_t* shared, int n, PrefixPlan o) {
  const int g = (int)blockIdx.x;
  auto edge = [&](int i) {
    const int b = cu_groups[i];
    return b < 0 ? 0 : b > a.B ? a.B : b;
  };
  auto row_of = [&](int b) {  // the first token row of sequence b, or of what lies behind the last
    if (b < a.B) return seq_rows(a.cu, b, a.T).first;
    const SeqRows last = seq_rows(a.cu, a.B - 1, a.T);
    return last.first + last.n;
  };
  const int cap = a.row_pages << a.page_shift;
  auto cover = [&](int b, int tokens, int group) {
    if (!o.entries) {
      o.skip[b] = tokens;
      return;
    }
    const SeqRows r = seq_rows(a.cu, b, a.T);
    const int len = a.lens[b];
    o.entries[b] = Kv8Entry{r.first, r.n, len < 0 ? 0 : len > cap ? cap : len, r.n ? tokens : 0, b, group, 0, 0};
  };
  if (g == n) {
    const int lo = edge(0), hi = edge(n);
    for (int b = (int)threadIdx.x; b < a.B; b += 256)
      if (b < lo || b >= hi) cover(b, 0, -1);
    if (threadIdx.x == 0 && !o.entries) o.cu[n] = row_of(hi);
    return;
  }
  const int b0 = edge(g), b1 = edge(g + 1);
  int most = shared[g], with = 0, from = 0x7FFFFFFF;  // from: the first sequence with queries
  for (int b = b0 + (int)threadIdx.x; b < b1; b += 256) {
    const SeqRows r = seq_rows(a.cu, b, a.T);
    if (r.n == 0) continue;
    const int len = a.lens[b] < cap ? a.lens[b] : cap;
    most = len - r.n < most ? len - r.n : most;
    from = b < from ? b : from;
    ++with;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const int other = __shfl_xor(most, d, 64), before = __shfl_xor(from, d, 64);
    most = other < most ? other : most;
    from = before < from ? before : from;
    with += __shfl_xor(with, d, 64);
  }
  __shared__ int part[4][3];
  if ((threadIdx.x & 63) == 0) {
    part[threadIdx.x >> 6][0] = most;
    part[threadIdx.x >> 6][1] = with;
    part[threadIdx.x >> 6][2] = from;
  }
  __syncthreads();
  with = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    most = part[i][0] < most ? part[i][0] : most;
    with += part[i][1];
    from = part[i][2] < from ? part[i][2] : from;
  }
  if (with == 0) from = 0;
  const int covered = kv8_covered(a, most, with);
  for (int b = b0 + (int)threadIdx.x; b < b1; b += 256) cover(b, covered, g);
  if (threadIdx.x == 0 && o.entries) {
    const int row0 = row_of(b0), end = b1 > b0 ? row_of(b1) : row0;
    o.entries[a.B + g] = Kv8Entry{row0, end > row0 ? end - row0 : 0, covered, 0, from, kIsGroup, 0, 0};
  } else if (threadIdx.x == 0) {
    o.cu[g] = row_of(b0);
    o.lens[g] = covered;
    o.row[g] = from;
  }
}

// The workspace: the plan's numbers, the first pass' sums (in one pass: the whole items of groups,
// then those of sequences), then the parts.
struct PrefixSpace {
  Kv8JointPlan joint;
  AttnPlans first, second;  // where it does not serve
  size_t acc, ml, own_acc, own_ml, rest, total;
};
PrefixSpace prefix_space(int64_t T, int64_t B, int Hkv, int G, int D, int64_t tokens, int64_t n) {
  auto round = [](size_t x) { return (x + 255) / 256 * 256; };
  PrefixSpace s;
  s.joint = kv8_joint_plan(T, B, n, Hkv, G, D, tokens, device_cu_count());
  const size_t sums = round((size_t)T * Hkv * G * D * 4), weights = round((size_t)T * Hkv * G * 8);
  s.acc = s.joint.items ? round((size_t)(B + n) * sizeof(Kv8Entry)) : round((size_t)(3 * n + 1 + B) * 4);
  s.ml = s.acc + sums;
  s.own_acc = s.ml + weights;
  s.own_ml = s.own_acc + (s.joint.items ? sums : 0);
  s.rest = s.own_ml + (s.joint.items ? weights : 0);
  if (s.joint.items) {
    s.total = s.rest + (size_t)(2 * s.joint.parts * Hkv * s.joint.slot_rows * (D + 2)) * sizeof(float);
  } else {
    s.first = attn_plans(T, n, Hkv, G, D, tokens);
    s.second = attn_plans(T, B, Hkv, G, D, tokens);
    const size_t x = attn_workspace(s.first, Hkv, D), y = attn_workspace(s.second, Hkv, D);
    s.total = s.rest + (x > y ? x : y);
  }
  return s;
}

}  // namespace
}  // namespace sgl

extern "C" {

size_t sgl_kv8_attn_workspace_size(int64_t T, int64_t B, int Hkv, int G, int D, int64_t max_tokens) {
  if (!sgl::attn_sizes_ok(T, B, Hkv, G, D, max_tokens)) return 0;
  return sgl::attn_workspace(sgl::attn_plans(T, B, Hkv, G, D, max_tokens), Hkv, D);
}

int sgl_kv8_attn(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype, int64_t T, int64_t B,
                 int Hkv, int G, int D, const int32_t* cu_tokens, const int32_t* lens, const int32_t* block_table,
                 int64_t row_pages, int page_size, int block, int64_t n_pages, const void* k_codes,
                 const void* v_codes, const float* k_scale, const float* v_scale, float softmax_scale, int causal,
                 int64_t window, const float* sink, void* out, void* workspace, size_t workspace_bytes,
                 sgl_stream_t stream) {
  return sgl_kv8_attn_first(q, q_token_stride, q_head_stride, dtype, T, B, Hkv, G, D, cu_tokens, lens, block_table,
                            row_pages, page_size, block, n_pages, k_codes, v_codes, k_scale, v_scale, softmax_scale,
                            causal, window, 0, sink, out, workspace, workspace_bytes, stream);
}

size_t sgl_kv8_attn_first_workspace_size(int64_t T, int64_t B, int Hkv, int G, int D, int64_t max_tokens,
                                         int64_t window, int64_t first) {
  if (!sgl::attn_sizes_ok(T, B, Hkv, G, D, max_tokens) || window < 0 || first < 0) return 0;
  return sgl::attn_workspace(
      sgl::attn_plans(T, B, Hkv, G, D, sgl::kv8_attn_reach(T, B, max_tokens, window, first), first > 0), Hkv, D);
}

int sgl_kv8_attn_first(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype, int64_t T, int64_t B,
                       int Hkv, int G, int D, const int32_t* cu_tokens, const int32_t* lens,
                       const int32_t* block_table, int64_t row_pages, int page_size, int block, int64_t n_pages,
                       const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale,
                       float softmax_scale, int causal, int64_t window, int64_t first, const float* sink, void* out,
                       void* workspace, size_t workspace_bytes, sgl_stream_t stream) {
  const sgl::AttnCall call = {q, q_token_stride, q_head_stride, dtype, T, B, Hkv, G, D, cu_tokens, lens, block_table,
                              row_pages, page_size, block, n_pages, k_codes, v_codes, k_scale, v_scale, softmax_scale,
                              causal, window, sink, out, workspace};
  sgl::Kv8AttnArgs a;
  bool nothing;
  SGL_REQUIRE(first >= 0 && (first == 0 || window > 0), "kv8_attn: first tokens (%lld) are for a window", (long long)first);
  int rc = sgl::attn_args(call, a, nothing);
  if (rc != SGL_OK || nothing) return rc;
  const int64_t tokens = row_pages * page_size, reach = sgl::kv8_attn_reach(T, B, tokens, window, first);
  a.first = a.window == 0 ? 0 : (int)(first < tokens ? first : tokens);
  const sgl::AttnPlans plans = sgl::attn_plans(T, B, Hkv, G, D, reach, first > 0);
  rc = sgl::check_workspace(workspace, workspace_bytes, sgl::attn_workspace(plans, Hkv, D));
  if (rc == SGL_OK) rc = sgl::check_plans(plans, tokens);
  if (rc != SGL_OK) return rc;
  sgl::launch_plans(a, dtype, plans, (hipStream_t)stream);
  return sgl::check_launch("kv8_attn");
}

size_t sgl_kv8_attn_shared_workspace_size(int64_t T, int64_t B, int Hkv, int G, int D, int64_t max_tokens,
                                          int64_t n_groups) {
  if (!sgl::attn_sizes_ok(T, B, Hkv, G, D, max_tokens) || n_groups < 1) return 0;
  return sgl::prefix_space(T, B, Hkv, G, D, max_tokens, n_groups).total;
}

int sgl_kv8_attn_shared(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype, int64_t T, int64_t B,
                        int Hkv, int G, int D, const int32_t* cu_tokens, const int32_t* lens,
                        const int32_t* block_table, int64_t row_pages, int page_size, int block, int64_t n_pages,
                        const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale,
                        float softmax_scale, int causal, const float* sink, int64_t n_groups,
                        const int32_t* cu_groups, const int32_t* shared, void* out, void* workspace,
                        size_t workspace_bytes, sgl_stream_t stream) {
  const sgl::AttnCall call = {q, q_token_stride, q_head_stride, dtype, T, B, Hkv, G, D, cu_tokens, lens, block_table,
                              row_pages, page_size, block, n_pages, k_codes, v_codes, k_scale, v_scale, softmax_scale,
                              causal, 0, sink, out, workspace};
  sgl::Kv8AttnArgs a;
  bool nothing;
  SGL_REQUIRE(n_groups >= 1 && n_groups <= (1 << 24), "kv8_attn: n_groups=%lld out of range", (long long)n_groups);
  int rc = sgl::attn_args(call, a, nothing);
  if (rc != SGL_OK || nothing) return rc;
  SGL_REQUIRE(cu_groups && shared, "kv8_attn: null pointer");
  const int64_t tokens = row_pages * page_size, n = n_groups;
  const sgl::PrefixSpace space = sgl::prefix_space(T, B, Hkv, G, D, tokens, n);
  const bool joint = space.joint.items != 0;
  rc = sgl::check_workspace(workspace, workspace_bytes, space.total);
  if (rc == SGL_OK && !joint) rc = sgl::check_plans(space.first, tokens);
  if (rc == SGL_OK && !joint) rc = sgl::check_plans(space.second, tokens);
  if (rc != SGL_OK) return rc;
  const int64_t items = space.joint.items + space.joint.group_items;
  SGL_REQUIRE_SUPPORTED(!joint || (items * ((tokens + 31) / 32 + sgl::kItemCost) < (1ll << 31) &&
                                   T * Hkv * G < (1ll << 31)),
                        "kv8_attn: %lld row tiles over %lld tokens are too many for one call", (long long)items,
                        (long long)tokens);
  char* base = (char*)workspace;
  sgl::PrefixPlan plan = {};
  if (joint) {
    plan.entries = (sgl::Kv8Entry*)base;
  } else {
    plan.cu = (int32_t*)base;
    plan.lens = plan.cu + n + 1;
    plan.row = plan.lens + n;
    plan.skip = plan.row + n;
  }
  a.ws_acc = (float*)(base + space.rest);
  a.prior_acc = (float*)(base + space.acc);
  a.prior_ml = (float*)(base + space.ml);
  const hipStream_t st = (hipStream_t)stream;
  const bool planned = !joint || !sgl::kv8_joint_alone(B, n);
  if (planned) sgl::kv8_prefix_kernel<<<(unsigned)(n + 1), 256, 0, st>>>(a, cu_groups, shared, (int)n, plan);
  if (joint) {
    const sgl::Kv8JointPlan& p = space.joint;
    a.B = (int)(B + n);
    a.groups = (int)n;
    a.group_rows = (int)p.group_rows;
    a.slot_rows = (int)p.slot_rows;
    a.parts = (int)p.parts;
    a.above = 0;
    a.upto = 0x7FFFFFFF;
    a.entries = planned ? plan.entries : nullptr;
    a.cu_groups = cu_groups;
    a.shared = shared;
    a.own_acc = (float*)(base + space.own_acc);
    a.own_ml = (float*)(base + space.own_ml);
    a.ws_ml = a.ws_acc + 2 * p.parts * Hkv * p.slot_rows * D;
    if (dtype == SGL_BF16)
      sgl::launch_joint<SGL_BF16>(a, p, st);
    else
      sgl::launch_joint<SGL_F16>(a, p, st);
    return sgl::check_launch("kv8_attn");
  }
  sgl::Kv8AttnArgs g = a;
  g.B = (int)n;
  g.cu = plan.cu;
  g.lens = plan.lens;
  g.table_row = plan.row;
  g.causal = false;
  g.sink = nullptr;
  g.raw = true;
  sgl::launch_plans(g, dtype, space.first, st);
  a.skip = plan.skip;
  sgl::launch_plans(a, dtype, space.second, st);
  return sgl::check_launch("kv8_attn");
}

}  // extern "C"
