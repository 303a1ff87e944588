// What the attention kernels over the 8-bit paged cache (kv8_attn.hip,
// kv8_prefill.hip) share: arguments, the order of the work, the merge of parts.
// Not part of the C ABI.
//
// A sequence's n queries and the G query heads of one kv head make n G rows
// (row r: query r / G, head r % G), cut into row tiles.  An item is (sequence,
// row tile, kv head); its keys are cut into key tiles.  Items follow each other
// by sequence, row tile, head; the key tiles of all items make one line, which
// the workgroups share evenly: each takes `per` tiles of it in order.  So a
// batch of ragged lengths keeps every CU as busy as an even one, and nothing on
// the host needs to know the lengths.  An item inside one workgroup is written
// out; of one that several share, each leaves its unnormalised sums, reference
// point and weight in the workspace (at most two such parts a workgroup, one at
// either end of its line), and the merge joins them in the order of the line.
#pragma once

#include "sgl_kv8.h"

namespace sgl {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;

struct Kv8AttnArgs {
  const uint16_t* q;
  int64_t qt, qh;  // elements between tokens, heads
  uint16_t* o;     // [T, Hkv G, D]
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int32_t *pages, *lens, *cu;
  const float* sink;  // [Hkv G] or null
  int64_t n_pages;
  int T, B, Hkv, G, D, row_pages, page_shift, block_shift;
  float c1;     // softmax scale in log2 units
  int window;   // keys a query sees, itself included; 0: all
  bool causal;
  int wgs;
  float* ws_acc;  // [2 wgs][row tile][D]
  float* ws_ml;   // [2 wgs][row tile][2]: reference point (log2 units), sum
};

struct Kv8Seq {
  int row0, n, len;  // first query row, queries, keys
  int tile0, tiles;  // key tiles: first, number (at least one, so that empty rows are written)
  int row_tiles;
};

template <int RT, int TT>
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8AttnArgs& a, int b) {
  const SeqRows r = seq_rows(a.cu, b, a.T);
  const int cap = a.row_pages << a.page_shift;
  int len = a.lens[b];
  len = len < 0 ? 0 : len > cap ? cap : len;
  int lo = 0;
  if (a.causal && a.window > 0) {
    const int64_t first = (int64_t)len - r.n - a.window + 1;
    lo = first > 0 ? (int)first : 0;
  }
  Kv8Seq s;
  s.row0 = r.first;
  s.n = r.n;
  s.len = len;
  s.tile0 = lo / TT;
  const int tiles = (len + TT - 1) / TT - s.tile0;
  s.tiles = tiles > 0 ? tiles : 1;
  s.row_tiles = (r.n * a.G + RT - 1) / RT;
  return s;
}

// Where something lies on the line.
struct Kv8Place {
  int b;       // sequence; B: behind the last
  int64_t before;  // key tiles of the sequences before
  int items;   // items of the sequences before
};

// The line's length.
template <int RT, int TT>
__device__ __forceinline__ int64_t kv8_total(const Kv8AttnArgs& a) {
  const int lane = threadIdx.x & 63;
  int64_t total = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    int c = 0;
    if (b0 + lane < a.B) {
      const Kv8Seq s = kv8_seq<RT, TT>(a, b0 + lane);
      c = s.tiles * s.row_tiles * a.Hkv;
    }
    total += __builtin_amdgcn_readlane(wave_incl_scan(c), 63);
  }
  return total;
}

// The sequence that holds tile x of the line (BY_ITEM: item x).
template <int RT, int TT, bool BY_ITEM>
__device__ __forceinline__ Kv8Place kv8_find(const Kv8AttnArgs& a, int64_t x) {
  const int lane = threadIdx.x & 63;
  Kv8Place at = {0, 0, 0};
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    int c = 0, k = 0;
    if (b0 + lane < a.B) {
      const Kv8Seq s = kv8_seq<RT, TT>(a, b0 + lane);
      k = s.row_tiles * a.Hkv;
      c = s.tiles * k;
    }
    const int ci = wave_incl_scan(c), ki = wave_incl_scan(k);
    const uint64_t past = __ballot(BY_ITEM ? at.items + ki > x : at.before + ci > x);
    if (past) {
      const int l = __builtin_ctzll(past);
      at.b = b0 + l;
      at.before += __builtin_amdgcn_readlane(ci, l) - __builtin_amdgcn_readlane(c, l);
      at.items += __builtin_amdgcn_readlane(ki, l) - __builtin_amdgcn_readlane(k, l);
      return at;
    }
    at.before += __builtin_amdgcn_readlane(ci, 63);
    at.items += __builtin_amdgcn_readlane(ki, 63);
  }
  at.b = a.B;
  return at;
}

template <int QT>
__device__ __forceinline__ uint32_t kv8_out2(float a, float b) {
  return pack2<QT>(a, b);
}

// Items that several workgroups share, one workgroup each: 256 threads.
template <int RT, int TT, int QT>
__global__ __launch_bounds__(256) void kv8_merge_kernel(const Kv8AttnArgs a) {
  const int64_t total = kv8_total<RT, TT>(a);
  const int64_t per = (total + a.wgs - 1) / a.wgs;
  const Kv8Place at = kv8_find<RT, TT, true>(a, (int64_t)blockIdx.x);
  if (at.b >= a.B) return;
  const Kv8Seq s = kv8_seq<RT, TT>(a, at.b);
  const int item = (int)blockIdx.x - at.items;
  const int64_t xs = at.before + (int64_t)item * s.tiles, xe = xs + s.tiles;
  const int wa = (int)(xs / per), wb = (int)((xe - 1) / per);
  if (wa == wb) return;
  const int rt = item / a.Hkv, head = item - rt * a.Hkv;
  const int rows = s.n * a.G - rt * RT;
  const int chunks = a.D >> 3;
  for (int i = threadIdx.x; i < RT * chunks; i += 256) {
    const int r = i / chunks, d = (i - r * chunks) << 3;
    if (r >= rows) return;
    const int row = rt * RT + r, t = row / a.G, h = head * a.G + (row - t * a.G);
    float M = -__builtin_huge_valf();
    for (int w = wa; w <= wb; ++w) M = __builtin_fmaxf(M, a.ws_ml[((int64_t)(2 * w + (w == wa)) * RT + r) * 2]);
    const float ref = M == -__builtin_huge_valf() ? 0.0f : M;
    float l = a.sink ? __builtin_amdgcn_exp2f(a.sink[h] * kLog2e - ref) : 0.0f;
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
    for (int w = wa; w <= wb; ++w) {
      const int64_t slot = (int64_t)(2 * w + (w == wa)) * RT + r;
      const float2 ml = *reinterpret_cast<const float2*>(a.ws_ml + slot * 2);
      const float4* p = reinterpret_cast<const float4*>(a.ws_acc + slot * a.D + d);
      const float4 x = p[0], y = p[1];
      const float f = __builtin_amdgcn_exp2f(ml.x - ref);
      l += ml.y * f;
      acc[0] += x.x * f; acc[1] += x.y * f; acc[2] += x.z * f; acc[3] += x.w * f;
      acc[4] += y.x * f; acc[5] += y.y * f; acc[6] += y.z * f; acc[7] += y.w * f;
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
#pragma unroll
    for (int v = 0; v < 8; ++v) acc[v] *= inv;
    *reinterpret_cast<uint4*>(a.o + ((int64_t)(s.row0 + t) * (a.Hkv * a.G) + h) * a.D + d) =
        make_uint4(kv8_out2<QT>(acc[0], acc[1]), kv8_out2<QT>(acc[2], acc[3]), kv8_out2<QT>(acc[4], acc[5]),
                   kv8_out2<QT>(acc[6], acc[7]));
  }
}

// kv8_prefill.hip: row tiles of 128.  plan.wgs == 0: a workgroup takes a whole item.
void launch_kv8_prefill(const Kv8AttnArgs& a, const Kv8AttnPlan& plan, int dtype, hipStream_t stream);

}  // namespace sgl
