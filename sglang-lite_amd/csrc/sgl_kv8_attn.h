// What the attention kernels over the 8-bit paged cache (kv8_attn.hip,
// kv8_prefill.hip) share: arguments, the order of the work, the merge of parts.
// Not part of the C ABI.
//
// A sequence's n queries and the G query heads of one kv head make n G rows
// (row r: query r / G, head r % G), cut into row tiles.  An item is (sequence,
// row tile, kv head); its keys are cut into key tiles.  For each kv head the key
// tiles of all items, one sequence after the other, make one line, which `parts`
// workgroups share evenly: so a batch of ragged lengths of single tokens keeps every CU as busy
// as an even one, and nothing on the host needs to know the lengths.  (Not so with chunks, whose
// row tiles each have the sequence's key tiles on the line, also those that none of its rows sees:
// a prompt of 8192 1030 us on shared lines, 560 with an item each.)  An item also
// takes kItemCost tiles' room on the line, for its start and end.  The
// workgroups of the same part of the lines, which read the same pages, run on
// one XCD at about the same time.
// An item inside one workgroup is written out; of one that several share, each
// leaves its unnormalised sums, reference point and weight in the workspace (at
// most two such parts a workgroup, one at either end of its stretch), and the
// merge joins them in the order of the line.
#pragma once

#include "sgl_kv8.h"

namespace sgl {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;

// The products take weights as f16, 2^kLift times what the reference point makes of them: an
// f16 reaches 2^16 above 1 but loses bits from 2^-14 on and is 0 from 2^-25 on, and small weights
// are all that a row has where the keys above them have no value.  So a key's weight keeps 11
// bits down to 2^-24 of the row's largest (each times its value's scale) and counts down to 2^-35
// of it, about 24 in the exponent of e.  2^kLift is in the exponent beside the value's scale, so it
// costs nothing but the room for a maximum to grow before a reference has to move.
constexpr float kLift = 10.0f, kUnlift = 0x1p-10f;

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
  int parts;      // workgroups of a kv head's line; 0: one workgroup an item
  int above, upto;  // takes the sequences of more than `above` rows a kv head, and up to `upto`
  float* ws_acc;  // [2 parts Hkv][row tile][D]
  float* ws_ml;   // [2 parts Hkv][row tile][2]: reference point (log2 units), sum
};

// Key tiles.  1 / 2 / 3 / 5, us: 32 sequences of 4 queries up to 6000 keys 49.3 / 48.2 / 46.1 /
// 47.2, 16 single ones up to 4000 25.6 / 24.8 / 23.3 / 23.5, 512 queries on 2000 57.0 / 55.2 / 51.8 / 53.8.
constexpr int kItemCost = 3;

// In the place of a granule's exponent (kLift + log2 of its value scale, -90 to 138): there is no
// such token; a scale of it is negative or not finite, which makes NaN of its keys and values;
// its values count as zero (NaN codes as NaN).  The last is for value scales below 2^-100, whose
// reciprocal times the weights of a long sequence would not fit fp32: no value of theirs reaches
// 2^-91.  The append writes 2^-100 at least.
constexpr float kNoToken = 1000.0f, kBadScale = 2000.0f, kNoValue = -91.0f;
__device__ __forceinline__ bool kv8_scale_ok(float s) { return s >= 0.0f && s < __builtin_huge_valf(); }
__device__ __forceinline__ float kv8_exponent(bool there, bool good, float vs) {
  return !there ? kNoToken : !good ? kBadScale : vs < 0x1p-100f ? kNoValue : __builtin_amdgcn_logf(vs) + kLift;
}

// A sequence as the line sees it.
struct Kv8Seq {
  int row0, n, len;  // first query row, queries, keys
  int tile0, tiles;  // key tiles: first, number (at least one, so that empty rows are written)
  int row_tiles;
};

template <int RT, int TT>
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8AttnArgs& a, int row0, int n, int len) {
  int lo = 0;
  if (a.causal && a.window > 0) {
    const int64_t first = (int64_t)len - n - a.window + 1;
    lo = first > 0 ? (int)first : 0;
  }
  Kv8Seq s;
  s.row0 = row0;
  s.n = n;
  s.len = len;
  s.tile0 = lo / TT;
  const int tiles = (len + TT - 1) / TT - s.tile0;
  s.tiles = tiles > 0 ? tiles : 1;
  s.row_tiles = (n * a.G + RT - 1) / RT;
  return s;
}

// 64 sequences from b0 on, one a lane.
struct Kv8Chunk {
  int b0, row0, n, len;
  int room, rooms;  // places on the line: of this sequence, of those up to and with it
  int rts;          // row tiles of the sequences up to and with it
};

template <int RT, int TT>
__device__ __forceinline__ Kv8Chunk kv8_chunk(const Kv8AttnArgs& a, int b0) {
  const int b = b0 + (int)(threadIdx.x & 63);
  Kv8Chunk c = {b0, 0, 0, 0, 0, 0, 0};
  int rts = 0;
  if (b < a.B) {
    const int len = a.lens[b], cap = a.row_pages << a.page_shift;
    const SeqRows r = seq_rows(a.cu, b, a.T);
    c.row0 = r.first;
    c.n = r.n;
    c.len = len < 0 ? 0 : len > cap ? cap : len;
    const Kv8Seq s = kv8_seq<RT, TT>(a, c.row0, c.n, c.len);
    const int rows = r.n * a.G;
    rts = rows > a.above && rows <= a.upto ? s.row_tiles : 0;
    c.room = rts * (s.tiles + kItemCost);
  }
  c.rooms = wave_incl_scan(c.room);
  c.rts = wave_incl_scan(rts);
  return c;
}

template <int RT, int TT>
__device__ __forceinline__ Kv8Seq kv8_lane(const Kv8AttnArgs& a, const Kv8Chunk& c, int l) {
  return kv8_seq<RT, TT>(a, __builtin_amdgcn_readlane(c.row0, l), __builtin_amdgcn_readlane(c.n, l),
                         __builtin_amdgcn_readlane(c.len, l));
}

// Length of a kv head's line; c: the batch's first 64 sequences.
template <int RT, int TT>
__device__ __forceinline__ int64_t kv8_total(const Kv8AttnArgs& a, const Kv8Chunk& c) {
  int64_t total = __builtin_amdgcn_readlane(c.rooms, 63);
  for (int b0 = 64; b0 < a.B; b0 += 64) total += __builtin_amdgcn_readlane(kv8_chunk<RT, TT>(a, b0).rooms, 63);
  return total;
}

// The sequence that holds place x of the line (BY_TILE: row tile x): lane `l` of
// chunk c, and what lies before the sequence.  l < 0: behind the last.
struct Kv8Place {
  int l;
  int64_t room;  // places before
  int64_t rts;   // row tiles before
};
template <int RT, int TT, bool BY_TILE>
__device__ __forceinline__ Kv8Place kv8_find(const Kv8AttnArgs& a, Kv8Chunk& c, int64_t x) {
  Kv8Place at = {-1, 0, 0};
  for (;;) {
    const uint64_t past = __ballot(BY_TILE ? at.rts + c.rts > x : at.room + c.rooms > x);
    if (past) {
      at.l = __builtin_ctzll(past);
      if (at.l > 0) {
        at.room += __builtin_amdgcn_readlane(c.rooms, at.l - 1);
        at.rts += __builtin_amdgcn_readlane(c.rts, at.l - 1);
      }
      return at;
    }
    at.room += __builtin_amdgcn_readlane(c.rooms, 63);
    at.rts += __builtin_amdgcn_readlane(c.rts, 63);
    if (c.b0 + 64 >= a.B) return at;
    c = kv8_chunk<RT, TT>(a, c.b0 + 64);
  }
}

// Workgroup of a kv head's part, and back: the heads of a part follow each other
// on one XCD (workgroups go round the eight in order; parts is a multiple of 8).
__device__ __forceinline__ int kv8_wg(const Kv8AttnArgs& a, int head, int part) {
  return ((part >> 3) * a.Hkv + head) * 8 + (part & 7);
}
__device__ __forceinline__ void kv8_wg_at(const Kv8AttnArgs& a, int wg, int* head, int* part) {
  const int k = wg >> 3, p = k / a.Hkv;
  *head = k - p * a.Hkv;
  *part = 8 * p + (wg & 7);
}

// A stretch of an item's key tiles that one workgroup takes.
struct Kv8Segment {
  Kv8Seq s;
  int b, rt;   // sequence, row tile
  int t0, t1;  // key tiles, from the item's first
};

// Walks over the segments of the places [x, end) of a line.
template <int RT, int TT>
struct Kv8Walk {
  Kv8Chunk c;
  int64_t x, end, base;
  int l;

  __device__ __forceinline__ bool start(const Kv8AttnArgs& a, int part) {
    c = kv8_chunk<RT, TT>(a, 0);
    const int64_t total = kv8_total<RT, TT>(a, c), per = (total + a.parts - 1) / a.parts;
    x = (int64_t)part * per;
    end = x + per < total ? x + per : total;
    if (x >= end) return false;
    const Kv8Place at = kv8_find<RT, TT, false>(a, c, x);
    base = at.room;
    l = at.l;
    return true;
  }
  // The next segment; false: none left.
  __device__ __forceinline__ bool next(const Kv8AttnArgs& a, Kv8Segment& g) {
    while (x < end) {
      const int room = __builtin_amdgcn_readlane(c.room, l);
      if (x >= base + room) {
        base += room;
        if (++l == 64) {
          if (c.b0 + 64 >= a.B) return false;
          c = kv8_chunk<RT, TT>(a, c.b0 + 64);
          l = 0;
        }
        continue;
      }
      g.s = kv8_lane<RT, TT>(a, c, l);
      g.b = c.b0 + l;
      const int size = g.s.tiles + kItemCost, off = (int)(x - base);
      g.rt = off / size;
      const int at = off - g.rt * size;
      const int64_t left = end - x;
      const int to = size - at < left ? size : at + (int)left;
      x += to - at;
      g.t0 = at > kItemCost ? at - kItemCost : 0;
      g.t1 = to - kItemCost;
      if (g.t1 > g.t0) return true;
    }
    return false;
  }
};

template <int QT>
__device__ __forceinline__ uint32_t kv8_out2(float a, float b) {
  return pack2<QT>(a, b);
}

// Item x of the batch (row tiles in order, the heads of each together) as one segment.
template <int RT, int TT>
__device__ __forceinline__ bool kv8_item(const Kv8AttnArgs& a, int64_t x, int* head, Kv8Segment& g) {
  const int64_t tile = x / a.Hkv;
  *head = (int)(x - tile * a.Hkv);
  Kv8Chunk c = kv8_chunk<RT, TT>(a, 0);
  const Kv8Place at = kv8_find<RT, TT, true>(a, c, tile);
  if (at.l < 0) return false;
  g.s = kv8_lane<RT, TT>(a, c, at.l);
  g.b = c.b0 + at.l;
  g.rt = (int)(tile - at.rts);
  g.t0 = 0;
  g.t1 = g.s.tiles;
  return true;
}

// The items that several workgroups share.  One wavefront a row (four a workgroup,
// RT / 4 workgroups an item): lane p has part p's reference and weight, and all lanes
// go over the parts' sums.
template <int RT, int TT, int QT>
__global__ __launch_bounds__(256) void kv8_merge_kernel(const Kv8AttnArgs a) {
  Kv8Chunk c = kv8_chunk<RT, TT>(a, 0);
  const int64_t total = kv8_total<RT, TT>(a, c), per = (total + a.parts - 1) / a.parts;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = blockIdx.x / (RT / 4);
  const int head = (int)(item % a.Hkv);
  const Kv8Place at = kv8_find<RT, TT, true>(a, c, item / a.Hkv);
  if (at.l < 0) return;
  const Kv8Seq s = kv8_lane<RT, TT>(a, c, at.l);
  const int rt = (int)(item / a.Hkv - at.rts);
  const int64_t xs = at.room + (int64_t)rt * (s.tiles + kItemCost) + kItemCost;
  const int pa = (int)(xs / per), pb = (int)((xs + s.tiles - 1) / per);
  const int r = 4 * (int)(blockIdx.x % (RT / 4)) + wave;
  if (pa == pb || r >= s.n * a.G - rt * RT) return;
  const int row = rt * RT + r, t = row / a.G, h = head * a.G + (row - t * a.G);
  const float NEG_INF = -__builtin_huge_valf();
  auto slot = [&](int p) { return (2 * (int64_t)kv8_wg(a, head, p) + (p == pa ? 1 : 0)) * RT + r; };

  // sums of 8 parts from p on, on their way while the references (or the last 8) are worked on
  const int d = 4 * lane;
  auto fetch = [&](int p, float4* x) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      x[k] = *reinterpret_cast<const float4*>(a.ws_acc + slot(p + k < pb ? p + k : pb) * a.D + (d < a.D ? d : 0));
  };
  float4 x[8];
  fetch(pa, x);
  float M = NEG_INF;
  for (int p = pa + lane; p <= pb; p += 64) M = __builtin_fmaxf(M, a.ws_ml[slot(p) * 2]);
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) M = __builtin_fmaxf(M, __shfl_xor(M, k, 64));
  const float ref = M == NEG_INF ? 0.0f : M;
  float l = 0.0f, acc[4] = {0, 0, 0, 0};
  for (int p0 = pa; p0 <= pb; p0 += 64) {
    float f = 0.0f;
    if (p0 + lane <= pb) {
      const float2 ml = *reinterpret_cast<const float2*>(a.ws_ml + slot(p0 + lane) * 2);
      f = __builtin_amdgcn_exp2f(ml.x - ref);
      l += ml.y * f;
    }
    const int n = pb - p0 < 63 ? pb - p0 + 1 : 64;
    for (int i = 0; i < n; i += 8) {
      float4 y[8];
      if (p0 + i + 8 <= pb) fetch(p0 + i + 8, y);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (i + k < n) {
          const float w = bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(f), i + k));
          acc[0] += x[k].x * w;
          acc[1] += x[k].y * w;
          acc[2] += x[k].z * w;
          acc[3] += x[k].w * w;
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = y[k];
    }
  }
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) l += __shfl_xor(l, k, 64);
  if (a.sink) l += __builtin_amdgcn_exp2f(a.sink[h] * kLog2e - ref);
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  if (d < a.D)
    *reinterpret_cast<uint2*>(a.o + ((int64_t)(s.row0 + t) * (a.Hkv * a.G) + h) * a.D + d) =
        make_uint2(kv8_out2<QT>(acc[0] * inv, acc[1] * inv), kv8_out2<QT>(acc[2] * inv, acc[3] * inv));
}

// kv8_prefill.hip: row tiles of kv8_chunk_rows(D).
void launch_kv8_prefill(const Kv8AttnArgs& a, const Kv8AttnPlan& plan, int dtype, hipStream_t stream);

}  // namespace sgl
