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
  int first;    // and the sequence's first tokens, which the window does not hide
  bool causal;
  int parts;      // workgroups of a kv head's line; 0: one workgroup an item
  int above, upto;  // takes the sequences of more than `above` rows a kv head, and up to `upto`
  float* ws_acc;  // [2 parts Hkv][row tile][D]
  float* ws_ml;   // [2 parts Hkv][row tile][2]: reference point (log2 units), sum
  // A common prefix in two passes: its groups are the sequences of the first, whose unnormalised
  // sums go to `prior` (`raw`); the second begins behind what they cover, and joins the two.
  const int32_t* table_row;  // first pass: the row of the block table of each group; null: its own
  const int32_t* skip;       // second pass: tokens that the first has covered; null: none
  float* prior_acc;          // [T Hkv G][D]
  float* prior_ml;           // [T Hkv G][2]
  bool raw;
  // In one: the sequences and behind them the groups on one line, `entries` of them B; whole
  // items go to `prior` (groups) and `own` (sequences).
  const struct Kv8Entry* entries;  // null: 64 at most, and each workgroup finds them by itself
  const int32_t *cu_groups, *shared;  // of the caller
  int groups, group_rows, slot_rows;  // of them; rows of a group's tile; of a part
  float *own_acc, *own_ml;
};

// A sequence or a group: its query rows, keys, the tokens in front that its group has covered, the
// row of the block table, its group (-1: none; kIsGroup: it is one).
struct __attribute__((aligned(16))) Kv8Entry {
  int row0, n, len, skip;
  int table_row, group, pad0, pad1;
};
constexpr int kIsGroup = -2;

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

// What a kernel is made for: plain calls; first tokens beside the window; either of two passes of a
// common prefix; its only one.  (In one kernel for all, the others cost plain calls 1 to 3 %.)
enum Kv8Mode { kPlain, kFirst, kShared, kJoint };
inline Kv8Mode kv8_mode(const Kv8AttnArgs& a) { return a.raw || a.skip ? kShared : a.first > 0 ? kFirst : kPlain; }

// A sequence as the line sees it.
struct Kv8Seq {
  int row0, n, len;  // first query row, queries, keys
  int tile0, tiles;  // key tiles: hidden ones in front, number (at least one, so that empty rows are written)
  int kept;          // tiles of the first tokens, which lie before the hidden ones
  int row_tiles;
  int skip;
  int table_row, group;

  // the key tile that tile i of the item is
  template <int MODE>
  __device__ __forceinline__ int tile(int i) const {
    return MODE == kFirst && i < kept ? i : i + tile0;
  }
};

template <int RT, int TT, int MODE>
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8AttnArgs& a, int row0, int n, int len, int skip, int group) {
  int lo = MODE == kShared || MODE == kJoint ? skip : 0;
  if (a.causal && a.window > 0) {
    const int64_t first = (int64_t)len - n - a.window + 1;
    lo = first > 0 ? (int)first : 0;
  }
  Kv8Seq s;
  s.row0 = row0;
  s.n = n;
  s.len = len;
  s.skip = skip;
  s.kept = MODE == kFirst ? (a.first + TT - 1) / TT : 0;
  s.tile0 = MODE != kFirst || lo / TT > s.kept ? lo / TT - s.kept : 0;
  const int tiles = (len + TT - 1) / TT - s.tile0;
  s.tiles = tiles > 0 ? tiles : 1;
  s.group = group;
  if (MODE == kJoint && group == kIsGroup)
    s.row_tiles = (n * a.G + a.group_rows - 1) / a.group_rows;
  else
    s.row_tiles = (n * a.G + RT - 1) / RT;
  return s;
}

// 64 sequences from b0 on, one a lane.
struct Kv8Chunk {
  int b0, row0, n, len, skip, table_row, group;
  int room, rooms;  // places on the line: of this sequence, of those up to and with it
  int rts;          // row tiles of the sequences up to and with it
};

// The chunk's places, once its sequences are there.
template <int RT, int TT, int MODE>
__device__ __forceinline__ void kv8_places(const Kv8AttnArgs& a, Kv8Chunk& c) {
  int rts = 0;
  if (c.b0 + (int)(threadIdx.x & 63) < a.B) {
    const Kv8Seq s = kv8_seq<RT, TT, MODE>(a, c.row0, c.n, c.len, c.skip, c.group);
    const int rows = c.n * a.G;
    // (a group that shares nothing has no part in the work)
    const bool none = c.len == 0 && ((MODE == kShared && a.raw) || (MODE == kJoint && c.group == kIsGroup));
    rts = rows > a.above && rows <= a.upto && !none ? s.row_tiles : 0;
    c.room = rts * (s.tiles + kItemCost);
  }
  c.rooms = wave_incl_scan(c.room);
  c.rts = wave_incl_scan(rts);
}

template <int RT, int TT, int MODE>
__device__ __forceinline__ Kv8Chunk kv8_chunk(const Kv8AttnArgs& a, int b0) {
  const int b = b0 + (int)(threadIdx.x & 63);
  Kv8Chunk c = {b0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  if (b < a.B) {
    if constexpr (MODE == kJoint) {
      const Kv8Entry e = a.entries[b];
      c.row0 = e.row0;
      c.n = e.n;
      c.len = e.len;
      c.skip = e.skip;
      c.table_row = e.table_row;
      c.group = e.group;
    } else {
      const int len = a.lens[b], cap = a.row_pages << a.page_shift;
      const SeqRows r = seq_rows(a.cu, b, a.T);
      c.row0 = r.first;
      c.n = r.n;
      c.len = len < 0 ? 0 : len > cap ? cap : len;
      if (MODE == kShared && a.skip) c.skip = a.skip[b];
    }
  }
  kv8_places<RT, TT, MODE>(a, c);
  return c;
}

// ---- a common prefix.  A group's queries all see the keys [0, covered), so the group is taken
// as one sequence of these keys, whose rows meet the keys' tiles together, and each of its sequences
// from there on.  `covered` is what the caller says, cut to whole pages and key tiles (of every
// kernel: 128 tokens), and to what lies before the first query (`most`) of each of the group's
// sequences that has any (`with` of them); 0 for a group of fewer than two such.  The pages are those of the
// first of these: of a sequence without queries neither its length nor its row of the block table is looked at.
constexpr int kPrefixTile = 128;
__device__ __forceinline__ int kv8_covered(const Kv8AttnArgs& a, int most, int with) {
  const int unit = kPrefixTile > (1 << a.page_shift) ? kPrefixTile : 1 << a.page_shift;
  return with < 2 || most < unit ? 0 : most & ~(unit - 1);
}

// Least of a wavefront by DPP moves, the same in every lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ int least_moved(int v) {
  const int o = __builtin_amdgcn_update_dpp(0x7FFFFFFF, v, CTRL, ROWS, 0xF, false);
  return o < v ? o : v;
}
__device__ __forceinline__ int wave_min(int v) {
  v = least_moved<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v = least_moved<0x112, 0xF>(v);
  v = least_moved<0x114, 0xF>(v);
  v = least_moved<0x118, 0xF>(v);
  v = least_moved<0x142, 0xA>(v);  // row_bcast 15
  v = least_moved<0x143, 0xC>(v);  // row_bcast 31
  return __builtin_amdgcn_readlane(v, 63);
}

// All of a line of up to 64 sequences and groups, without a launch before that plans it: a sequence
// or group a lane, each group's covered tokens from its lanes.
template <int RT, int TT>
__device__ __forceinline__ Kv8Chunk kv8_joint_chunk(const Kv8AttnArgs& a) {
  const int lane = (int)(threadIdx.x & 63), sequences = a.B - a.groups;
  Kv8Chunk c = {0, 0, 0, 0, 0, lane, -1, 0, 0, 0};
  int e0 = 0, e1 = 0, most = 0;  // of a group: its sequences, what the caller says
  if (lane < sequences) {
    const int len = a.lens[lane], cap = a.row_pages << a.page_shift;
    const SeqRows r = seq_rows(a.cu, lane, a.T);
    c.row0 = r.first;
    c.n = r.n;
    c.len = len < 0 ? 0 : len > cap ? cap : len;
  } else if (lane < a.B) {
    auto edge = [&](int b) { return b < 0 ? 0 : b > sequences ? sequences : b; };
    e0 = edge(a.cu_groups[lane - sequences]);
    e1 = edge(a.cu_groups[lane - sequences + 1]);
    most = a.shared[lane - sequences];
  }
  const int behind = __builtin_amdgcn_readlane(c.row0 + c.n, sequences - 1);  // the last one's rows
  for (int l = sequences; l < a.B; ++l) {
    const int b0 = __builtin_amdgcn_readlane(e0, l), b1 = __builtin_amdgcn_readlane(e1, l);
    const bool in = lane >= b0 && lane < b1, counts = in && c.n > 0;
    const int least = wave_min(counts ? c.len - c.n : 0x7FFFFFFF), said = __builtin_amdgcn_readlane(most, l);
    const uint64_t with = __ballot(counts);
    const int covered = kv8_covered(a, least < said ? least : said, __builtin_popcountll(with));
    if (in) {
      c.skip = c.n ? covered : 0;
      c.group = l - sequences;
    }
    const int first = b0 < sequences ? __builtin_amdgcn_readlane(c.row0, b0) : behind;
    const int end = b1 < sequences ? __builtin_amdgcn_readlane(c.row0, b1) : behind;
    if (lane == l) {
      c.row0 = first;
      c.n = b1 > b0 && end > first ? end - first : 0;
      c.len = covered;
      c.table_row = with ? __builtin_ctzll(with) : 0;
      c.group = kIsGroup;
    }
  }
  kv8_places<RT, TT, kJoint>(a, c);
  return c;
}
// the line's first chunk
template <int RT, int TT, int MODE>
__device__ __forceinline__ Kv8Chunk kv8_first_chunk(const Kv8AttnArgs& a) {
  if constexpr (MODE == kJoint) {
    if (!a.entries) return kv8_joint_chunk<RT, TT>(a);
  }
  return kv8_chunk<RT, TT, MODE>(a, 0);
}

template <int RT, int TT, int MODE>
__device__ __forceinline__ Kv8Seq kv8_lane(const Kv8AttnArgs& a, const Kv8Chunk& c, int l) {
  Kv8Seq s = kv8_seq<RT, TT, MODE>(a, __builtin_amdgcn_readlane(c.row0, l), __builtin_amdgcn_readlane(c.n, l),
                                   __builtin_amdgcn_readlane(c.len, l),
                                   MODE == kShared || MODE == kJoint ? __builtin_amdgcn_readlane(c.skip, l) : 0,
                                   MODE == kJoint ? __builtin_amdgcn_readlane(c.group, l) : 0);
  if (MODE == kJoint) s.table_row = __builtin_amdgcn_readlane(c.table_row, l);
  return s;
}

// Length of a kv head's line; c: the batch's first 64 sequences.
template <int RT, int TT, int MODE>
__device__ __forceinline__ int64_t kv8_total(const Kv8AttnArgs& a, const Kv8Chunk& c) {
  int64_t total = __builtin_amdgcn_readlane(c.rooms, 63);
  for (int b0 = 64; b0 < a.B; b0 += 64) total += __builtin_amdgcn_readlane(kv8_chunk<RT, TT, MODE>(a, b0).rooms, 63);
  return total;
}

// The sequence that holds place x of the line (BY_TILE: row tile x): lane `l` of
// chunk c, and what lies before the sequence.  l < 0: behind the last.
struct Kv8Place {
  int l;
  int64_t room;  // places before
  int64_t rts;   // row tiles before
};
template <int RT, int TT, int MODE, bool BY_TILE>
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
    c = kv8_chunk<RT, TT, MODE>(a, c.b0 + 64);
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
template <int RT, int TT, int MODE>
struct Kv8Walk {
  Kv8Chunk c;
  int64_t x, end, base;
  int l;

  __device__ __forceinline__ bool start(const Kv8AttnArgs& a, int part) {
    c = kv8_first_chunk<RT, TT, MODE>(a);
    const int64_t total = kv8_total<RT, TT, MODE>(a, c), per = (total + a.parts - 1) / a.parts;
    x = (int64_t)part * per;
    end = x + per < total ? x + per : total;
    if (x >= end) return false;
    const Kv8Place at = kv8_find<RT, TT, MODE, false>(a, c, x);
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
          c = kv8_chunk<RT, TT, MODE>(a, c.b0 + 64);
          l = 0;
        }
        continue;
      }
      g.s = kv8_lane<RT, TT, MODE>(a, c, l);
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

// What is to be done with the sums of a row (reference point M, sum) that all of its keys have
// gone into: the first pass keeps them; the others join the first's, take the sink
// and divide.  `own` and `before` are the factors of the sums and of the prior ones.
struct Kv8Join {
  float own, before;
  bool prior;
};
template <int MODE>
__device__ __forceinline__ Kv8Join kv8_join(const Kv8AttnArgs& a, const Kv8Seq& s, int64_t at, int h, float M, float sum) {
  const float NEG_INF = -__builtin_huge_valf();
  Kv8Join j = {1.0f, 0.0f, MODE == kShared && s.skip > 0};
  float top = M;
  float2 ml = make_float2(NEG_INF, 0.0f);
  if (j.prior) {
    ml = *reinterpret_cast<const float2*>(a.prior_ml + 2 * at);
    top = __builtin_fmaxf(M, ml.x);
  }
  const float ref = top == NEG_INF ? 0.0f : top;
  if (j.prior) {
    j.own = __builtin_amdgcn_exp2f(M - ref);
    j.before = __builtin_amdgcn_exp2f(ml.x - ref);
    sum = sum * j.own + ml.y * j.before;
  }
  if (a.sink) sum += __builtin_amdgcn_exp2f(a.sink[h] * kLog2e - ref);
  const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
  j.own *= inv;
  j.before *= inv;
  return j;
}
// four of the row's sums
template <int MODE>
__device__ __forceinline__ float4 kv8_joined(const Kv8AttnArgs& a, const Kv8Join& j, int64_t at, int d, float4 y) {
  y = make_float4(y.x * j.own, y.y * j.own, y.z * j.own, y.w * j.own);
  if (MODE == kShared && j.prior) {
    const float4 p = *reinterpret_cast<const float4*>(a.prior_acc + at * a.D + d);
    y = make_float4(y.x + p.x * j.before, y.y + p.y * j.before, y.z + p.z * j.before, y.w + p.w * j.before);
  }
  return y;
}

// Item x of the batch (row tiles in order, the heads of each together) as one segment.
template <int RT, int TT, int MODE>
__device__ __forceinline__ bool kv8_item(const Kv8AttnArgs& a, int64_t x, int* head, Kv8Segment& g) {
  const int64_t tile = x / a.Hkv;
  *head = (int)(x - tile * a.Hkv);
  Kv8Chunk c = kv8_chunk<RT, TT, MODE>(a, 0);
  const Kv8Place at = kv8_find<RT, TT, MODE, true>(a, c, tile);
  if (at.l < 0) return false;
  g.s = kv8_lane<RT, TT, MODE>(a, c, at.l);
  g.b = c.b0 + at.l;
  g.rt = (int)(tile - at.rts);
  g.t0 = 0;
  g.t1 = g.s.tiles;
  return true;
}

// The items that several workgroups share.  One wavefront a row (four a workgroup,
// RT / 4 workgroups an item): lane p has part p's reference and weight, and all lanes
// go over the parts' sums.
template <int RT, int TT, int QT, int MODE>
__global__ __launch_bounds__(256) void kv8_merge_kernel(const Kv8AttnArgs a) {
  Kv8Chunk c = kv8_chunk<RT, TT, MODE>(a, 0);
  const int64_t total = kv8_total<RT, TT, MODE>(a, c), per = (total + a.parts - 1) / a.parts;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = blockIdx.x / (RT / 4);
  const int head = (int)(item % a.Hkv);
  const Kv8Place at = kv8_find<RT, TT, MODE, true>(a, c, item / a.Hkv);
  if (at.l < 0) return;
  const Kv8Seq s = kv8_lane<RT, TT, MODE>(a, c, at.l);
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
  if (d >= a.D) return;
  const int64_t out = (int64_t)(s.row0 + t) * (a.Hkv * a.G) + h;
  float4 y = make_float4(acc[0], acc[1], acc[2], acc[3]);
  if (MODE == kShared && a.raw) {
    *reinterpret_cast<float4*>(a.prior_acc + out * a.D + d) = y;
    if (lane == 0) *reinterpret_cast<float2*>(a.prior_ml + 2 * out) = make_float2(M, l);
    return;
  }
  y = kv8_joined<MODE>(a, kv8_join<MODE>(a, s, out, h, M, l), out, d, y);
  *reinterpret_cast<uint2*>(a.o + out * a.D + d) = make_uint2(kv8_out2<QT>(y.x, y.y), kv8_out2<QT>(y.z, y.w));
}

// The rows of a batch whose sequences and groups were on one line: a row's own parts and its
// group's, one wavefront a row (a token's head).
template <int RT, int TT, int QT>
__global__ __launch_bounds__(256) void kv8_joint_merge_kernel(const Kv8AttnArgs a) {
  const int lane = threadIdx.x & 63, sequences = a.B - a.groups;
  const uint32_t heads = (uint32_t)(a.Hkv * a.G);
  const uint32_t out = 4 * blockIdx.x + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tok = (int)(out / heads), h = (int)(out - (uint32_t)tok * heads);
  if (tok >= a.T) return;
  const int head = h / a.G;
  // one walk over the line: the row's sequence, behind all of them its group, and the length
  // (fewer than 2^31 places: the call is checked for it)
  Kv8Seq s, gs;
  int entry = -1, total = 0, room = 0, before = 0;
  bool found = false;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const Kv8Chunk c = b0 == 0 ? kv8_first_chunk<RT, TT, kJoint>(a) : kv8_chunk<RT, TT, kJoint>(a, b0);
    const uint64_t mine = __ballot(b0 + lane < sequences && tok >= c.row0 && tok < c.row0 + c.n);
    auto rooms_before = [&](int l) { return total + (l > 0 ? __builtin_amdgcn_readlane(c.rooms, l - 1) : 0); };
    if (!found && mine) {
      const int l = __builtin_ctzll(mine);
      found = true;
      s = kv8_lane<RT, TT, kJoint>(a, c, l);
      room = rooms_before(l);
      if (s.skip > 0 && s.group >= 0) entry = sequences + s.group;
    }
    if (entry >= b0 && entry < b0 + 64) {
      gs = kv8_lane<RT, TT, kJoint>(a, c, entry - b0);
      before = rooms_before(entry - b0);
    }
    total += __builtin_amdgcn_readlane(c.rooms, 63);
  }
  if (!found) return;
  const uint32_t per = ((uint32_t)total + a.parts - 1) / a.parts;
  const int row = (tok - s.row0) * a.G + h - head * a.G;

  // the row's sums: parts [pa, pb] of its item, or (one workgroup took it whole) by its place in the output
  struct Source {
    const float *acc, *ml;  // whole
    int pa, n, r;
  };
  auto source = [&](int first, const Kv8Seq& q, uint32_t tile, int r, const float* acc, const float* ml) {
    const uint32_t x = (uint32_t)first + tile * (uint32_t)(q.tiles + kItemCost) + kItemCost;
    Source o = {acc + (int64_t)out * a.D, ml + 2 * (int64_t)out, (int)(x / per), 0, r};
    o.n = (int)((x + q.tiles - 1) / per) - o.pa + 1;
    return o;
  };
  const Source own = source(room, s, (uint32_t)row / RT, row % RT, a.own_acc, a.own_ml);
  Source shared = own;
  shared.n = 0;
  if (entry >= 0) {
    const int gr = (tok - gs.row0) * a.G + h - head * a.G;
    const uint32_t tile = (uint32_t)gr / (uint32_t)a.group_rows;
    // (a group without keys has no place on the line: falling cu_groups could name one)
    if (gr >= 0 && gr < gs.n * a.G && gs.len > 0)
      shared = source(before, gs, tile, gr - (int)tile * a.group_rows, a.prior_acc, a.prior_ml);
  }
  const int n = own.n + shared.n;
  auto slot = [&](const Source& o, int i) {
    return (2 * (int64_t)kv8_wg(a, head, o.pa + i) + (i == 0 ? 1 : 0)) * a.slot_rows + o.r;
  };
  auto acc_at = [&](int i) {
    const bool mine = i < own.n;
    const Source& o = mine ? own : shared;
    return o.n == 1 ? o.acc : a.ws_acc + slot(o, mine ? i : i - own.n) * a.D;
  };
  auto ml_at = [&](int i) {
    const bool mine = i < own.n;
    const Source& o = mine ? own : shared;
    return *reinterpret_cast<const float2*>(o.n == 1 ? o.ml : a.ws_ml + slot(o, mine ? i : i - own.n) * 2);
  };

  const float NEG_INF = -__builtin_huge_valf();
  const int d = 4 * lane, dl = d < a.D ? d : 0;
  auto fetch = [&](int i, float4* x) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = *reinterpret_cast<const float4*>(acc_at(i + k < n ? i + k : n - 1) + dl);
  };
  float4 x[8];
  fetch(0, x);
  float M = NEG_INF;
  for (int i = lane; i < n; i += 64) M = __builtin_fmaxf(M, ml_at(i).x);
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) M = __builtin_fmaxf(M, __shfl_xor(M, k, 64));
  const float ref = M == NEG_INF ? 0.0f : M;
  float l = 0.0f, acc[4] = {0, 0, 0, 0};
  for (int i0 = 0; i0 < n; i0 += 64) {
    float f = 0.0f;
    if (i0 + lane < n) {
      const float2 ml = ml_at(i0 + lane);
      f = __builtin_amdgcn_exp2f(ml.x - ref);
      l += ml.y * f;
    }
    const int m = n - i0 < 64 ? n - i0 : 64;
    for (int i = 0; i < m; i += 8) {
      float4 y[8];
      if (i0 + i + 8 < n) fetch(i0 + i + 8, y);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (i + k < m) {
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
    *reinterpret_cast<uint2*>(a.o + (int64_t)out * a.D + d) =
        make_uint2(kv8_out2<QT>(acc[0] * inv, acc[1] * inv), kv8_out2<QT>(acc[2] * inv, acc[3] * inv));
}

// kv8_prefill.hip: row tiles of kv8_chunk_rows(D).
void launch_kv8_prefill(const Kv8AttnArgs& a, const Kv8AttnPlan& plan, int dtype, hipStream_t stream);

}  // namespace sgl
