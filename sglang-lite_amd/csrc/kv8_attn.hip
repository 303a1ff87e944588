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

// DP: head dim rounded up to 64, 128 or 256; NC: 16-row column tiles
// SPLIT: workgroups share the lines, else a workgroup takes a whole item
template <int DP, int NC, int QT, bool SPLIT>
__global__ __launch_bounds__(64 * kWaves, DP == 64 ? 2 : 1) void kv8_attn_few_kernel(const Kv8AttnArgs a) {
  constexpr int RT = 16 * NC, KI = DP / 64, C = DP / 16, W = C / 4;
  __shared__ __align__(16) float sAcc[kWaves][16][DP + 4];
  __shared__ float sM[kWaves][16], sL[kWaves][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, g = lane >> 4;
  const float NEG_INF = -__builtin_huge_valf();

  int head, part = 0;
  Kv8Walk<RT, kTile> walk;
  Kv8Segment seg;
  if constexpr (SPLIT) {
    kv8_wg_at(a, (int)blockIdx.x, &head, &part);
    if (!walk.start(a, part)) return;
  } else {
    if (!kv8_item<RT, kTile>(a, (int64_t)blockIdx.x, &head, seg)) return;
  }
  for (bool more = SPLIT ? walk.next(a, seg) : true; more; more = SPLIT ? walk.next(a, seg) : false) {
    const Kv8Seq& s = seg.s;
    const int b = seg.b, rt = seg.rt, t0 = seg.t0, t1 = seg.t1;
    const int rows = s.n * a.G - rt * RT;  // valid rows of the tile (may be more than RT)

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
      hi[c] = !live ? 0 : a.causal ? pos + 1 : s.len;
      lo[c] = a.causal && a.window > 0 ? pos - a.window + 1 : 0;
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
    if (a.causal) {
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

    const int32_t* table = a.pages + (int64_t)b * a.row_pages;
    const int pmask = (1 << a.page_shift) - 1;
    const int first = (s.tile0 + t0) * kTile + 32 * wave;
    int stop = (s.tile0 + t1) * kTile;
    stop = stop < s.len ? stop : s.len;
    const int steps = first < stop ? (stop - first + kTile - 1) / kTile : 0;  // step i: tokens first + i kTile on

    // Pages and scales of 32 steps at a time: lane l has granule l & 1 of step l >> 1.
    // Loaded a batch ahead, so that no step waits for its table entry.
    struct Batch {
      int page;  // 0 where there is none
      float ks, vs;
      bool ok;
    };
    auto load_pages = [&](int batch) __attribute__((always_inline)) {
      Batch o;
      const int t = first + (32 * batch + (lane >> 1)) * kTile + 16 * (lane & 1);
      const int page = table[(t < s.len ? t : s.len - 1) >> a.page_shift];
      o.ok = t < s.len && page >= 0 && page < a.n_pages;
      o.page = o.ok ? page : 0;
      return o;
    };
    auto load_scales = [&](int batch, Batch& o) __attribute__((always_inline)) {
      const int t = first + (32 * batch + (lane >> 1)) * kTile + 16 * (lane & 1);
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
        const int spot = (first + i * kTile + 16 * u) & pmask;
        const int64_t row = ((((int64_t)page * a.Hkv + head) << a.page_shift) + spot) * a.D;
        const uint8_t* kp = a.kc + row;
        const uint8_t* vp = a.vc + row;
#pragma unroll
        for (int k = 0; k < KI; ++k) r.k[u][k] = ld16_stream(kp + (uint32_t)kd[k]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint8_t* at = vp + j * a.D + (uint32_t)vd;
          if constexpr (W == 1) {
            r.v[4 * u + j][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(at));
          } else if constexpr (W == 2) {
            const u2v y = __builtin_nontemporal_load(reinterpret_cast<const u2v*>(at));
            r.v[4 * u + j][0] = y.x;
            r.v[4 * u + j][1] = y.y;
          } else {
            const uint4 y = ld16_stream(at);
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
      const int tok = first + at * kTile, l0 = 2 * (at & 31);
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
      const bool plain = tok + 32 <= all_hi && tok >= all_lo && ok == 3;
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
            if (key < hi[c] && key >= lo[c] && key < s.len && ((here >> (i >> 2)) & 1u)) seen[c] |= 1u << i;
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
        sM[wave][m] = m_run[c];
        sL[wave][m] = l;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < C; j += 4)
          *reinterpret_cast<float4*>(&sAcc[wave][m][C * (4 * g + i) + j]) =
              make_float4(acc[c][j][i], acc[c][j + 1][i], acc[c][j + 2][i], acc[c][j + 3][i]);
      __syncthreads();
      const int chunks = a.D >> 3;
      for (int i = threadIdx.x; i < 16 * chunks; i += 64 * kWaves) {
        const int n = i / chunks, d = (i - n * chunks) << 3, r = 16 * c + n;
        if (r >= rows) break;
        float M = NEG_INF;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = __builtin_fmaxf(M, sM[w][n]);
        const float ref = M == NEG_INF ? 0.0f : M;
        float sum = 0.0f, y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float f = __builtin_amdgcn_exp2f(sM[w][n] - ref);
          sum += sL[w][n] * f;
#pragma unroll
          for (int v = 0; v < 8; ++v) y[v] += sAcc[w][n][d + v] * (f * kUnlift);
        }
        if (whole) {
          const int row = rt * RT + r, t = row / a.G, h = head * a.G + (row - t * a.G);
          if (a.sink) sum += __builtin_amdgcn_exp2f(a.sink[h] * kLog2e - ref);
          const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
#pragma unroll
          for (int v = 0; v < 8; ++v) y[v] *= inv;
          *reinterpret_cast<uint4*>(a.o + ((int64_t)(s.row0 + t) * (a.Hkv * a.G) + h) * a.D + d) =
              make_uint4(kv8_out2<QT>(y[0], y[1]), kv8_out2<QT>(y[2], y[3]), kv8_out2<QT>(y[4], y[5]),
                         kv8_out2<QT>(y[6], y[7]));
        } else {
          float4* out = reinterpret_cast<float4*>(a.ws_acc + (slot * RT + r) * a.D + d);
          out[0] = make_float4(y[0], y[1], y[2], y[3]);
          out[1] = make_float4(y[4], y[5], y[6], y[7]);
          if (d == 0) *reinterpret_cast<float2*>(a.ws_ml + (slot * RT + r) * 2) = make_float2(M, sum);
        }
      }
    }
  }
}

template <int DP, int NC, int QT>
void launch_few(const Kv8AttnArgs& a, int64_t items, hipStream_t st) {
  if (a.parts == 0) {
    kv8_attn_few_kernel<DP, NC, QT, false><<<(unsigned)items, 64 * kWaves, 0, st>>>(a);
    return;
  }
  kv8_attn_few_kernel<DP, NC, QT, true><<<a.parts * a.Hkv, 64 * kWaves, 0, st>>>(a);
  kv8_merge_kernel<16 * NC, kTile, QT><<<(unsigned)(items * 4 * NC), 256, 0, st>>>(a);
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

}  // namespace
}  // namespace sgl

extern "C" {

size_t sgl_kv8_attn_workspace_size(int64_t T, int64_t B, int Hkv, int G, int D, int64_t max_tokens) {
  if (T < 0 || B < 0 || Hkv < 1 || G < 1 || D < 16 || max_tokens < 0) return 0;
  size_t bytes = 0;
  for (const sgl::Kv8AttnPlan& p : {sgl::kv8_attn_plan(T, B, Hkv, G, D, max_tokens, sgl::device_cu_count()),
                                    sgl::kv8_attn_rest(T, B, Hkv, G, D, max_tokens, sgl::device_cu_count())}) {
    const size_t b = sgl::kv8_attn_workspace(p, Hkv, D);
    bytes = b > bytes ? b : bytes;
  }
  return bytes;
}

int sgl_kv8_attn(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype, int64_t T, int64_t B,
                 int Hkv, int G, int D, const int32_t* cu_tokens, const int32_t* lens, const int32_t* block_table,
                 int64_t row_pages, int page_size, int block, int64_t n_pages, const void* k_codes,
                 const void* v_codes, const float* k_scale, const float* v_scale, float softmax_scale, int causal,
                 int64_t window, const float* sink, void* out, void* workspace, size_t workspace_bytes,
                 sgl_stream_t stream) {
  SGL_REQUIRE(dtype == SGL_BF16 || dtype == SGL_F16, "kv8_attn: dtype %d (bf16 or f16)", dtype);
  const int rc = sgl::kv8_check_cache("kv8_attn", Hkv, D, page_size, block, n_pages, row_pages);
  if (rc != SGL_OK) return rc;
  SGL_REQUIRE(G >= 1 && (int64_t)G * Hkv <= 65536, "kv8_attn: G=%d query heads for each of %d kv heads", G, Hkv);
  SGL_REQUIRE(T >= 0 && B >= 0 && B <= (1 << 24) && T * G < (1ll << 31), "kv8_attn: T=%lld B=%lld out of range",
              (long long)T, (long long)B);
  SGL_REQUIRE(cu_tokens || T == B, "kv8_attn: without cu_tokens every sequence has one token (T=%lld, B=%lld)",
              (long long)T, (long long)B);
  SGL_REQUIRE(window >= 0 && (causal || window == 0), "kv8_attn: a window (%lld) is for causal attention",
              (long long)window);
  SGL_REQUIRE(softmax_scale > 0.0f && softmax_scale < 1e30f, "kv8_attn: softmax_scale must be positive");
  if (T == 0 || B == 0) return SGL_OK;
  SGL_REQUIRE(q && lens && block_table && k_codes && v_codes && k_scale && v_scale && out, "kv8_attn: null pointer");
  SGL_REQUIRE(sgl::aligned(q, 16) && q_token_stride % 8 == 0 && q_head_stride % 8 == 0,
              "kv8_attn: q and its strides must be 16-byte aligned");
  SGL_REQUIRE(sgl::aligned(k_codes, 16) && sgl::aligned(v_codes, 16) && sgl::aligned(out, 16),
              "kv8_attn: misaligned cache or output");
  // one launch, or (chunks and few rows in one batch) two, one after the other on the same workspace
  const int64_t tokens = row_pages * page_size;
  const sgl::Kv8AttnPlan plans[2] = {sgl::kv8_attn_plan(T, B, Hkv, G, D, tokens, sgl::device_cu_count()),
                                     sgl::kv8_attn_rest(T, B, Hkv, G, D, tokens, sgl::device_cu_count())};
  for (const sgl::Kv8AttnPlan& p : plans) {
    const size_t need = sgl::kv8_attn_workspace(p, Hkv, D);
    if (need && (!workspace || workspace_bytes < need)) {
      sgl::set_error("kv8_attn: workspace of %zu bytes, needs %zu", workspace ? workspace_bytes : 0, need);
      return SGL_ERR_WORKSPACE;
    }
    SGL_REQUIRE_SUPPORTED(p.items * ((tokens + 31) / 32 + sgl::kItemCost) < (1ll << 31) &&
                              p.items * p.row_tile / 4 < (1ll << 31),
                          "kv8_attn: %lld row tiles over %lld tokens are too many for one call", (long long)p.items,
                          (long long)tokens);
  }
  SGL_REQUIRE(sgl::aligned(workspace, 16), "kv8_attn: workspace must be 16-byte aligned");
  sgl::Kv8AttnArgs a;
  a.q = (const uint16_t*)q;
  a.qt = q_token_stride;
  a.qh = q_head_stride;
  a.o = (uint16_t*)out;
  a.kc = (const uint8_t*)k_codes;
  a.vc = (const uint8_t*)v_codes;
  a.ks = k_scale;
  a.vs = v_scale;
  a.pages = block_table;
  a.lens = lens;
  a.cu = cu_tokens;
  a.sink = sink;
  a.n_pages = n_pages;
  a.T = (int)T;
  a.B = (int)B;
  a.Hkv = Hkv;
  a.G = G;
  a.D = D;
  a.row_pages = (int)row_pages;
  a.page_shift = __builtin_ctz((unsigned)page_size);
  a.block_shift = __builtin_ctz((unsigned)block);
  a.c1 = softmax_scale * sgl::kLog2e;
  a.window = window >= tokens ? 0 : (int)window;  // (as long as the table: all keys)
  a.causal = causal != 0;
  a.ws_acc = (float*)workspace;
  for (const sgl::Kv8AttnPlan& p : plans) {
    if (p.items == 0) continue;
    if (dtype == SGL_BF16)
      sgl::launch_attn<SGL_BF16>(a, p, (hipStream_t)stream);
    else
      sgl::launch_attn<SGL_F16>(a, p, (hipStream_t)stream);
  }
  return sgl::check_launch("kv8_attn");
}

}  // extern "C"
