// attention_prefix.hip - attention of a batch whose sequences share a prefix of keys:
//
//   out = softmax(scale q [Kp; Ki]^T) [Vp; Vi],  lse = log sum exp(scale q [Kp; Ki]^T)
//
// for tokens q of sequence i, the prefix Kp, Vp and the sequence's own padded cache Ki,
// Vi. Every token sees the whole prefix. Running maximum, sum and output of a row over
// any set of keys join with those over any other (attention.hip), so there are two ways:
//
// Few rows per sequence (single tokens): the prefix is read once for the rows of all
// sequences, 128 of them per workgroup, cut into pieces over the GPU; so are the own
// caches, each for its own rows; a second kernel joins a row's pieces in order.
// What that reads is the floor: the prefix once, not once per sequence (one token of 16
// sequences behind 131072 keys, 56 heads over 8: 144 us, 4.5 TB/s in the first kernel, 7.5 in the second).
//
// Many rows per sequence: a workgroup's 128 rows walk the prefix and then the own cache
// in one pass. The prefix comes out of the caches, since the matrix units, not the keys, are
// what bounds it (878 tokens of four sequences behind 12605, 56 heads: 1.3 ms, 1.04 PFLOP/s).
// Few rows are walked too where there are few keys, for a kernel less.
//
// The softmax weights are rounded to the inputs' type for the product with v. At most 32 rows of a
// piece keep the rest of that rounding as a second number, so that the output's own rounding is all
// that is left. Other walks and pieces of more rows do without: their outputs' error against 64 bits is 1.40 times
// as large (bf16: 2.3e-3 of their size, of which rounding the output alone is 1.66e-3). The second number
// in those pieces too was measured: one token of 32 sequences behind 12605, 43 -> 47 us; of 16 behind
// 131072, 56 heads over 8, 143 -> 164; of 48, 40 heads over 8, 247 -> 295; 4 tokens of 16 behind 12605, 52 -> 67.
#include "lr_attention.h"
#include "lr_pieces.h"
#include "lr_runtime.h"

namespace lr {
namespace {

constexpr int kMaxPieces = 256;   // of a cache, and of the prefix
constexpr int kMaxCuts = 8;       // of the rows that a walk leaves behind its rounds

struct PrefixArgs {
  const uint16_t *q, *pk, *pv, *k, *v;
  uint16_t* out;
  float* lse;            // or null
  float* part;           // o [parts][dim], then (exponent, l, exact l, sees keys) [parts]
  int64_t qt, qh, qb;    // strides of a token, a head, a sequence, in elements
  int64_t pkt, pkh, pvt, pvh;
  int64_t kt, kh, kb;
  int64_t vt, vh, vb;
  const int32_t* lengths;   // valid keys of the own caches, or null
  int n, q_rows, k_rows, prefix;
  int heads, kv_heads, group;
  int causal;
  float c;               // scale * log2(e)
  int seq_tiles;         // tiles of 128 rows of a sequence
  int all_tiles;         // and of all sequences' rows together
  int places;            // workgroups per key head (pieces); 0: more sequences than a list holds
  int shares;            // most pieces of the prefix
  int own;               // most pieces of the own caches
  int piece;             // least tiles of 64 keys of a piece
  int whole, left, cuts; // walk: workgroups for all keys of their rows; those cut into `cuts`
};

__device__ __forceinline__ int own_keys(const PrefixArgs& p, int i) { return keys_of(p.lengths, i, p.k_rows); }
__device__ __forceinline__ int key_tiles(int keys) { return (int)((uint32_t)(keys + kKeys - 1) / kKeys); }

// How prefix and caches are cut: pieces of `size` tiles of 64 keys, the smallest for
// which all of them have a place. Every wave works it out from the lengths by itself.
struct Cut {
  int size, shared, prefix;   // tiles of a piece of a cache, and of the prefix; pieces of that one
  Pieces own;
  __device__ __forceinline__ explicit Cut(const PrefixArgs& p) {
    const int tiles = key_tiles(p.prefix);
    auto shared_of = [&](int size) __attribute__((always_inline)) { return max(size, ceil_div(tiles, p.shares)); };
    size = p.piece;
    if (p.places) {
      own.load(p.lengths, p.n, p.k_rows, kKeys);
      auto taken = [&](int size) __attribute__((always_inline)) {
        return own.count(size) * (float)p.seq_tiles + (float)(ceil_div(tiles, shared_of(size)) * p.all_tiles);
      };
      // From an even share up in steps, which end at the latest where every cache is one piece
      // (lr_attention_prefix gives as many places).
      size = max(max(size, ceil_div(key_tiles(p.k_rows), kMaxPieces)), (int)(taken(1) / (float)p.places));
      while (taken(size) > (float)p.places) size += max(1, size >> 4);
    }
    size = __builtin_amdgcn_readfirstlane(size);
    prefix = ceil_div(tiles, max(1, __builtin_amdgcn_readfirstlane(shared_of(size))));
    shared = Pieces::even(tiles, prefix);
  }
  // What has piece `place` of the caches: the sequence (-1: none) and its first piece.
  __device__ __forceinline__ void find(const PrefixArgs& p, int place, int& seq, int& first) const {
    if (p.places) own.find(p.n, size, place, seq, first);
    else seq = first = place < p.n ? place : -1;   // a piece each
  }
  // Each sequence's first piece and how many there are, and behind them the pieces of the prefix,
  // by one wave for the kernel that joins them.
  __device__ __forceinline__ void publish(const PrefixArgs& p, int2* table) const {
    const int lane = threadIdx.x & 63;
    int before = 0;
    if (p.places) {
#pragma unroll
      for (int g = 0; g < kListed / 64; ++g) {
        if (g >= own.groups) continue;
        const int n = ceil_div(own.tiles[g], size), upto = wave_prefix_sum(n);
        if (64 * g + lane < p.n) table[64 * g + lane] = make_int2(before + upto - n, n);
        before += __builtin_amdgcn_readlane(upto, 63);
      }
    } else {
      for (int i = lane; i < p.n; i += 64) table[i] = make_int2(i, own_keys(p, i) > 0);
    }
    if (lane == 0) table[p.n] = make_int2(prefix, 0);
  }
};

// The rows of a part of the prefix, of all sequences, come before those of the own pieces.
__device__ __forceinline__ int64_t own_part(const PrefixArgs& p, int piece) {
  const int64_t each = (int64_t)p.q_rows * p.heads;
  return ((int64_t)p.shares * p.n + piece) * each;
}
__device__ __forceinline__ int64_t all_parts(const PrefixArgs& p) { return own_part(p, p.own); }
// Behind the parts: which pieces a sequence has (Cut::publish).
template <int D>
__device__ __forceinline__ int2* pieces_of(const PrefixArgs& p) {
  return reinterpret_cast<int2*>(p.part + all_parts(p) * (D + 4));
}

// A sequence's rows 128 * tile .. and the own keys that they see.
struct OwnRows {
  int kn, rows, r0, sure, tiles;   // tiles: of the keys that any of them sees
  __device__ __forceinline__ OwnRows(const PrefixArgs& p, int seq, int tile) {
    kn = own_keys(p, seq);
    rows = p.q_rows * p.group;
    r0 = tile * kRows;
    sure = kn;
    int any = kn;
    if (p.causal) {
      const int last = min(r0 + kRows, rows) - 1;
      any = min(kn, max(0, kn - p.q_rows + (int)((uint32_t)last / (uint32_t)p.group) + 1));
      sure = min(kn, max(0, kn - p.q_rows + (int)((uint32_t)r0 / (uint32_t)p.group) + 1));
    }
    tiles = key_tiles(any);
  }
};

struct Row {
  int tok, head, seen;   // token (of the sequence or of all), head, own keys that it sees
  __device__ __forceinline__ Row(const PrefixArgs& p, int r, int rows, int hd, int kn) {
    const int rc = min(r, rows - 1);
    tok = (int)((uint32_t)rc / (uint32_t)p.group);
    head = hd * p.group + (rc - tok * p.group);
    seen = p.causal ? min(kn, max(0, kn - p.q_rows + tok + 1)) : kn;
  }
};

__device__ __forceinline__ OneCache own_cache(const PrefixArgs& p, int seq, int hd, const OwnRows& w, int seen) {
  return {p.k + seq * p.kb + hd * p.kh, p.v + seq * p.vb + hd * p.vh, p.kt, p.vt, w.kn, w.sure, seen};
}
__device__ __forceinline__ OneCache prefix_cache(const PrefixArgs& p, int hd) {
  return {p.pk + hd * p.pkh, p.pv + hd * p.pvh, p.pkt, p.pvt, p.prefix, p.prefix, p.prefix};
}

// attend for at most 32 rows, the same for all waves: what counts is the stream of keys. A wave
// takes 32 keys of each 128 by itself, through LDS of its own: they are all read into
// registers before they are worked on, and the next ones are on their way meanwhile, so that the
// whole workgroup's LDS is in flight (twice what the tiles of attend have) and no wave waits
// for another. Weights are kept as a rounded number and its rest, as there. The waves' rows
// are joined in LDS at the end, in their order: wave w is left with columns 16 w .. of each 64
// of the lane's row (D / 8 of o, in all of its D / 2), l and the exponent. (16 sequences of 40
// key heads behind 8192: 59 us, 4.4 TB/s; 68 with the tiles of attend.)
template <typename T, int D, class Keys>
__device__ __forceinline__ void attend_few(char* smem, float2* stats, const Keys& keys, const uint16_t* qrow, const float c,
                                           const int t0, const int t1, float& l, float& off, float (&mine)[D / 8]) {
  typedef typename Mfma<T>::V V8;
  constexpr int ROW = 2 * D, CH = ROW / 16, RPB = 256 / ROW, PAIRS = ROW / 32, KD = D / 16, DB = D / 32;
  constexpr int HALF = 32 * ROW, DMAS = HALF / 1024;   // a wave's keys, its values behind them
  static_assert(4 * 2 * HALF == kTileBytes<D>, "LDS");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int half = lane >> 5, col = lane & 31;
  char* const ks = smem + wave * 2 * HALF;
  char* const vs = ks + HALF;
  V8 q[KD];
#pragma unroll
  for (int d = 0; d < KD; ++d) q[d] = *reinterpret_cast<const V8*>(qrow + 16 * d + 8 * half);
  // The 16 bytes of a tile that this lane fetches.
  auto offset = [&](int i, uint32_t stride) __attribute__((always_inline)) {
    const int at = i * 64 + lane, row = at / CH, ch = at % CH ^ (row / RPB % PAIRS) * 2;
    return row * stride * 2 + ch * 16;
  };
  uint32_t koff[DMAS], voff[DMAS];
  if constexpr (Keys::kOneStride) {
#pragma unroll
    for (int i = 0; i < DMAS; ++i) {
      koff[i] = offset(i, (uint32_t)keys.stride(0, 0));
      voff[i] = offset(i, (uint32_t)keys.stride(0, 1));
    }
  }
  auto issue = [&](int s) {   // half s % 2 of tile s / 2; keys past the last read as zero
    const int t = s >> 1, left = min(32, keys.left(t) - 32 * (s & 1));
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const int64_t stride = keys.stride(t, v);
      const __amdgpu_buffer_rsrc_t r = row_rsrc(keys.at(t, v) + (left > 0 ? 32 * (s & 1) * stride : 0),
                                                left > 0 ? ((int64_t)(left - 1) * stride + D) * 2 : 0);
#pragma unroll
      for (int i = 0; i < DMAS; ++i)
        dma16(r, (v ? vs : ks) + i * 1024, Keys::kOneStride ? (v ? voff[i] : koff[i]) : offset(i, (uint32_t)stride));
    }
  };
  v16f o[DB];
  float m = -INFINITY, unused = 0.0f;
  l = off = 0.0f;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
  const int i16 = lane & 15, vr = 4 * half + (i16 >> 2);
  const int s1 = 2 * t1;
  int s = 2 * t0 + wave;
  if (s < s1) issue(s);
#pragma unroll 1
  for (; s < s1; s += 4) {
    __builtin_amdgcn_s_waitcnt(0x70 | 0xf00);   // vmcnt(0): this wave's keys and values are there
    asm volatile("" ::: "memory");
    V8 kf[KD], vf[2][DB];
#pragma unroll
    for (int d = 0; d < KD; ++d)
      kf[d] = *reinterpret_cast<const V8*>(ks + col * ROW + ((2 * d + half) ^ (col / RPB % PAIRS) * 2) * 16);
#pragma unroll
    for (int kc = 0; kc < 2; ++kc)
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const int ch = 4 * d + 2 * ((lane >> 4) & 1) + (i16 >> 1 & 1), r0 = 16 * kc + vr, r1 = r0 + 8;
        vf[kc][d] = tr_pair<V8>(vs + r0 * ROW + (ch ^ (r0 / RPB % PAIRS) * 2) * 16 + (i16 & 1) * 8,
                                vs + r1 * ROW + (ch ^ (r1 / RPB % PAIRS) * 2) * 16 + (i16 & 1) * 8);
      }
    __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): and in registers
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if (s + 4 < s1) issue(s + 4);
    v16f sc = {};
#pragma unroll
    for (int d = 0; d < KD; ++d) sc = Mfma<T>::mul(kf[d], q[d], sc);
    if (!keys.whole(s >> 1)) {
      const int lim = keys.limit(s >> 1) - keys.first(s >> 1) - 32 * (s & 1) - 4 * half;
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = 8 * (e >> 2) + (e & 3) < lim ? sc[e] : -INFINITY;
    }
    float x = sc[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) x = fmaxf(x, sc[e]);
    off = move_max<DB, false>(max_with_partner(x), m, l, unused, o, c, Mfma<T>::kShift);
#pragma unroll
    for (int kc = 0; kc < 2; ++kc) {
      uint4 hi, lo;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * kc + 2 * w], c, -off));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * kc + 2 * w + 1], c, -off));
        const uint32_t h = Mfma<T>::pack(p0, p1);
        set_word(hi, w, h);
        set_word(lo, w, Mfma<T>::pack(p0 - Mfma<T>::first(h), p1 - Mfma<T>::second(h)));
        l += p0 + p1;
      }
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        o[d] = Mfma<T>::mul(vf[kc][d], __builtin_bit_cast(V8, hi), o[d]);
        o[d] = Mfma<T>::mul(vf[kc][d], __builtin_bit_cast(V8, lo), o[d]);
      }
    }
  }
  // (Nothing is on its way to the LDS: the last keys have been waited for.)
  l = add_partner(l);
  __syncthreads();
  float* const parts = reinterpret_cast<float*>(smem);   // [wave][D / 2][lane]
  stats[wave * 64 + lane] = make_float2(off, l);
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) parts[(wave * (D / 2) + 16 * d + e) * 64 + lane] = o[d][e];
  __syncthreads();
  float2 st[4];
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    st[w] = stats[w * 64 + lane];
    if (st[w].y != 0.0f) top = fmaxf(top, st[w].x);
  }
  off = top == -INFINITY ? 0.0f : top;
  l = 0.0f;
#pragma unroll
  for (int i = 0; i < D / 8; ++i) mine[i] = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (st[w].y == 0.0f) continue;
    const float f = __builtin_amdgcn_exp2f(st[w].x - off);
    l += f * st[w].y;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) mine[i] += f * parts[(w * (D / 2) + wave * (D / 8) + i) * 64 + lane];
  }
}

// One piece of the prefix or of a cache for at most 128 rows.
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void prefix_pieces(PrefixArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[kTileBytes<D> + 256 * 8];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int half = lane >> 5, col = lane & 31;
  // All key heads of the same keys, which lie side by side, come first.
  const int hds = p.kv_heads, item = (int)(blockIdx.x / (uint32_t)hds), hd = (int)(blockIdx.x - item * hds);
  const Cut cut(p);
  if (blockIdx.x == 0 && wave == 0) cut.publish(p, pieces_of<D>(p));
  OneCache keys;
  int t0, t1, rows, r0, r;   // r: the lane's row
  int64_t part, qoff;
  bool sees, few;
  if (item < cut.prefix * p.all_tiles) {
    // The row tiles of a piece lie side by side, so that they share its keys in a cache.
    const int piece = (int)((uint32_t)item / (uint32_t)p.all_tiles);
    rows = p.n * p.q_rows * p.group;
    r0 = (item - piece * p.all_tiles) * kRows;
    few = rows - r0 <= 32;
    r = r0 + (few ? 0 : wave * 32) + col;
    const Row row(p, r, rows, hd, 0);
    const int seq = (int)((uint32_t)row.tok / (uint32_t)p.q_rows);
    qoff = seq * p.qb + (row.tok - seq * p.q_rows) * p.qt + row.head * p.qh;
    keys = prefix_cache(p, hd);
    t0 = piece * cut.shared;
    t1 = min(key_tiles(p.prefix), t0 + cut.shared);
    part = ((int64_t)piece * p.n * p.q_rows + row.tok) * p.heads + row.head;
    sees = true;
  } else {
    const int place = item - cut.prefix * p.all_tiles, piece = (int)((uint32_t)place / (uint32_t)p.seq_tiles);
    int seq, first;
    cut.find(p, piece, seq, first);
    if (seq < 0) return;
    const OwnRows w(p, seq, place - piece * p.seq_tiles);
    rows = w.rows;
    r0 = w.r0;
    few = rows - r0 <= 32;
    r = r0 + (few ? 0 : wave * 32) + col;
    const Row row(p, r, rows, hd, w.kn);
    qoff = seq * p.qb + row.tok * p.qt + row.head * p.qh;
    keys = own_cache(p, seq, hd, w, row.seen);
    const int all = key_tiles(w.kn), size = p.places ? Pieces::even(all, ceil_div(all, cut.size)) : all;
    t0 = min(w.tiles, (piece - first) * size);
    t1 = min(w.tiles, t0 + size);
    part = own_part(p, piece) + (int64_t)row.tok * p.heads + row.head;
    sees = row.seen > t0 * kKeys;
  }
  float* const po = p.part + part * D;
  float4* const stat = reinterpret_cast<float4*>(p.part + all_parts(p) * D) + part;
  float l, off;
  if (few) {
    float o[D / 8];
    attend_few<T, D>(smem, reinterpret_cast<float2*>(smem + kTileBytes<D>), keys, p.q + qoff, p.c, t0, t1, l, off, o);
    if (r >= rows) return;
    if (half == 0 && wave == 0) *stat = make_float4(off, l, l, sees);
    if (l == 0.0f) return;   // left out of the join by its l
#pragma unroll
    for (int g = 0; g < D / 32; ++g) {
      const int at = wave * (D / 32) + g;   // of the lane's D / 8 groups of four columns
      *reinterpret_cast<float4*>(po + 32 * (at / 4) + 8 * (at % 4) + 4 * half) =
          make_float4(o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]);
    }
    return;
  }
  v16f o[D / 32];
  float m, exact;
  attend<T, D, false, true>(smem, keys, p.q + qoff, p.c, t0, t1, r0 + wave * 32 >= rows, m, l, exact, off, o);
  l = add_partner(l);
  exact = add_partner(exact);
  if (r >= rows) return;
  if (half == 0) *stat = make_float4(off, l, exact, sees);
  if (l == 0.0f) return;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(po + 32 * d + 8 * g + 4 * half) =
          make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
}

constexpr float kLn2 = 0.69314718055994531f;
constexpr int kMaxParts = 2 * kMaxPieces;

// Joins a row's pieces of the prefix and of its cache: weights 2^(exponent - the largest). A
// workgroup per row: D / 4 threads hold a part's columns, and the groups of them take every
// G-th part, then are added in order, so that the result does not depend on timing.
template <typename T, int D>
__global__ __launch_bounds__(256) void prefix_join(PrefixArgs p) {
  const int64_t row = blockIdx.x;
  const int each = p.q_rows * p.heads, seq = (int)(blockIdx.x / (uint32_t)each);
  const int2 mine = pieces_of<D>(p)[seq];
  const int shared = pieces_of<D>(p)[p.n].x, n = shared + mine.y;
  const int64_t own = own_part(p, mine.x) + (row - (int64_t)seq * each);
  auto at = [&](int i) __attribute__((always_inline)) {
    return i < shared ? row + (int64_t)i * p.n * each : own + (int64_t)(i - shared) * each;
  };
  const float* const part = p.part;
  const float4* const stats = reinterpret_cast<const float4*>(p.part + all_parts(p) * D);
  constexpr int LANES = D / 4, G = 256 / LANES, NV = kMaxParts / 64;
  __shared__ float weight[kMaxParts];
  __shared__ float4 sums[G][LANES];
  const int t = threadIdx.x, lane = t & 63, x = t % LANES, g = t / LANES;
  // Every wave finds the maximum and the sums by itself.
  float4 v[NV];
  float top = -INFINITY, seen = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    v[i] = 64 * i + lane < n ? stats[at(64 * i + lane)] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (v[i].y != 0.0f) top = fmaxf(top, v[i].x);
    seen = fmaxf(seen, v[i].w);
  }
  top = wave_max(top);
  float l = 0.0f, exact = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const float w = v[i].y != 0.0f ? __builtin_amdgcn_exp2f(v[i].x - top) : 0.0f;
    weight[64 * i + lane] = w;   // the same value from each wave
    l += w * v[i].y;
    exact += w * v[i].z;
  }
  l = wave_tree_sum(l);
  exact = wave_tree_sum(exact);
  seen = wave_max(seen);
  __syncthreads();
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  constexpr int BATCH = 4;   // loads in flight
  for (int s0 = g; s0 < n; s0 += BATCH * G) {
    float4 y[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (s0 + i * G < n) y[i] = *reinterpret_cast<const float4*>(part + at(s0 + i * G) * D + 4 * x);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const float w = s0 + i * G < n ? weight[s0 + i * G] : 0.0f;
      if (w == 0.0f) continue;   // y was not written where the part had no keys
      o.x += w * y[i].x;
      o.y += w * y[i].y;
      o.z += w * y[i].z;
      o.w += w * y[i].w;
    }
  }
  sums[g][x] = o;
  __syncthreads();
  if (g != 0) return;
#pragma unroll
  for (int i = 1; i < G; ++i) {
    const float4 y = sums[i][x];
    o.x += y.x;
    o.y += y.y;
    o.z += y.z;
    o.w += y.w;
  }
  const float inv = l == 0.0f ? (seen != 0.0f ? NAN : 0.0f) : 1.0f / l;
  *reinterpret_cast<uint2*>(p.out + row * D + 4 * x) =
      make_uint2(Mfma<T>::pack(o.x * inv, o.y * inv), Mfma<T>::pack(o.z * inv, o.w * inv));
  if (p.lse && x == 0) p.lse[row] = l == 0.0f ? -INFINITY : kLn2 * (top + __builtin_amdgcn_logf(exact));
}

// The prefix, then the own cache. (Both sides of a choice are values: chosen between by
// address, the two would have to lie in memory.)
__device__ __forceinline__ int64_t either(bool first, int64_t a, int64_t b) { return first ? a : b; }
struct TwoCaches {
  OneCache a, b;
  int tiles;   // of a
  __device__ __forceinline__ int64_t stride(int t, int is_v) const {
    return is_v ? either(t < tiles, a.vt, b.vt) : either(t < tiles, a.kt, b.kt);
  }
  __device__ __forceinline__ const uint16_t* at(int t, int is_v) const {
    const int64_t base = is_v ? either(t < tiles, (int64_t)a.v, (int64_t)b.v) : either(t < tiles, (int64_t)a.k, (int64_t)b.k);
    return reinterpret_cast<const uint16_t*>(base) + (int64_t)first(t) * stride(t, is_v);
  }
  __device__ __forceinline__ int left(int t) const { return (int)either(t < tiles, a.kn, b.kn) - first(t); }
  __device__ __forceinline__ bool whole(int t) const { return first(t) + kKeys <= (int)either(t < tiles, a.sure, b.sure); }
  __device__ __forceinline__ int first(int t) const { return (t < tiles ? t : t - tiles) * kKeys; }
  __device__ __forceinline__ int limit(int t) const { return (int)either(t < tiles, a.seen, b.seen); }
  static constexpr bool kOneStride = false;
};

// What a workgroup of the walk has: a head's rows, of a sequence.
struct WalkItem {
  int hd, seq, tile;
  __device__ __forceinline__ WalkItem(const PrefixArgs& p, uint32_t id) {
    const uint32_t tiles = (uint32_t)(p.n * p.seq_tiles);
    hd = (int)(id / tiles);
    const int at = (int)(id - hd * tiles);
    seq = (int)((uint32_t)at / (uint32_t)p.seq_tiles);
    tile = at - seq * p.seq_tiles;
  }
};

// The first `whole` workgroups walk all keys of their rows. Those that would be left for a round
// of their own are cut into `cuts` runs of keys instead, joined by a second kernel.
template <typename T, int D, bool LSE>
__global__ __launch_bounds__(256, 2) void prefix_walk(PrefixArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[kTileBytes<D>];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int half = lane >> 5, col = lane & 31;
  // Each XCD takes a contiguous run of the heads' tiles, so that its L2 serves a head's
  // prefix to them all.
  const uint32_t whole = (uint32_t)p.whole, pid = blockIdx.x, per = whole >> 3, rest = whole & 7, xcd = pid & 7;
  const bool cut = pid >= whole;
  const uint32_t run = cut ? (pid - whole) / (uint32_t)p.cuts : 0, piece = cut ? pid - whole - run * p.cuts : 0;
  const WalkItem it(p, cut ? whole + run
                           : (xcd < rest ? xcd * (per + 1) : rest * (per + 1) + (xcd - rest) * per) + (pid >> 3));
  const OwnRows w(p, it.seq, it.tile);
  const int r = w.r0 + wave * 32 + col;
  const Row row(p, r, w.rows, it.hd, w.kn);
  const TwoCaches keys = {prefix_cache(p, it.hd), own_cache(p, it.seq, it.hd, w, row.seen), key_tiles(p.prefix)};
  const uint16_t* const q = p.q + it.seq * p.qb + row.tok * p.qt + row.head * p.qh;
  v16f o[D / 32];
  float m, l, exact, off;
  const bool idle = w.r0 + wave * 32 >= w.rows;
  const int tiles = keys.tiles + w.tiles, size = cut ? ceil_div(tiles, p.cuts) : tiles;
  const int t0 = min(tiles, (int)piece * size), t1 = min(tiles, t0 + size);
  attend<T, D, false, LSE>(smem, keys, q, p.c, t0, t1, idle, m, l, exact, off, o);
  l = add_partner(l);
  if (LSE) exact = add_partner(exact);
  if (r >= w.rows) return;
  const bool sees = p.prefix + row.seen > 0;
  if (cut) {
    const int64_t part = ((int64_t)run * p.cuts + piece) * kRows + wave * 32 + col;
    const int64_t parts = (int64_t)p.left * p.cuts * kRows;
    if (half == 0) reinterpret_cast<float4*>(p.part + parts * D)[part] = make_float4(off, l, LSE ? exact : l, sees);
    if (l == 0.0f) return;   // left out of the join by its l
    float* const po = p.part + part * D;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(po + 32 * d + 8 * g + 4 * half) =
            make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
    return;
  }
  const int64_t to = ((int64_t)it.seq * p.q_rows + row.tok) * p.heads + row.head;
  if (LSE && half == 0) p.lse[to] = l == 0.0f ? -INFINITY : kLn2 * (off + __builtin_amdgcn_logf(exact));
  const float inv = l == 0.0f ? (sees ? NAN : 0.0f) : 1.0f / l;
  uint16_t* const po = p.out + to * D;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<uint2*>(po + 32 * d + 8 * g + 4 * half) =
          make_uint2(Mfma<T>::pack(o[d][4 * g] * inv, o[d][4 * g + 1] * inv),
                     Mfma<T>::pack(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv));
}

// At most 32 rows per sequence and key head: all keys of them, without pieces and joins.
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void prefix_walk_few(PrefixArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[kTileBytes<D> + 256 * 8];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5;
  const int seq = (int)(blockIdx.x / (uint32_t)p.kv_heads), hd = (int)(blockIdx.x - seq * p.kv_heads), r = lane & 31;
  const OwnRows w(p, seq, 0);
  const Row row(p, r, w.rows, hd, w.kn);
  const TwoCaches keys = {prefix_cache(p, hd), own_cache(p, seq, hd, w, row.seen), key_tiles(p.prefix)};
  float l, off, o[D / 8];
  attend_few<T, D>(smem, reinterpret_cast<float2*>(smem + kTileBytes<D>), keys, p.q + seq * p.qb + row.tok * p.qt + row.head * p.qh,
                   p.c, 0, keys.tiles + w.tiles, l, off, o);
  if (r >= w.rows) return;
  const int64_t to = ((int64_t)seq * p.q_rows + row.tok) * p.heads + row.head;
  if (p.lse && half == 0 && wave == 0) p.lse[to] = l == 0.0f ? -INFINITY : kLn2 * (off + __builtin_amdgcn_logf(l));
  const float inv = l == 0.0f ? (p.prefix + row.seen > 0 ? NAN : 0.0f) : 1.0f / l;
#pragma unroll
  for (int g = 0; g < D / 32; ++g) {
    const int at = wave * (D / 32) + g;   // of the lane's D / 8 groups of four columns
    *reinterpret_cast<uint2*>(p.out + to * D + 32 * (at / 4) + 8 * (at % 4) + 4 * half) =
        make_uint2(Mfma<T>::pack(o[4 * g] * inv, o[4 * g + 1] * inv), Mfma<T>::pack(o[4 * g + 2] * inv, o[4 * g + 3] * inv));
  }
}

// Joins the cut workgroups' rows, as prefix_join does: a wave per row, and all of its at most
// eight parts at once.
template <typename T, int D>
__global__ __launch_bounds__(256) void walk_join(PrefixArgs p) {
  constexpr int LANES = D / 4, G = 64 / LANES, PER = kMaxCuts / G;
  const int lane = threadIdx.x & 63, x = lane % LANES, g = lane / LANES;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int run = (int)(id / kRows), at0 = (int)(id % kRows);
  const WalkItem it(p, (uint32_t)(p.whole + run));
  const int rows = p.q_rows * p.group, r = it.tile * kRows + at0;
  if (r >= rows) return;
  const Row row(p, r, rows, it.hd, 0);
  const int64_t to = ((int64_t)it.seq * p.q_rows + row.tok) * p.heads + row.head;
  const float4* const stats = reinterpret_cast<const float4*>(p.part + (int64_t)p.left * p.cuts * kRows * D);
  const int64_t first = (int64_t)run * p.cuts * kRows + at0;
  float4 v[kMaxCuts], y[PER];
#pragma unroll
  for (int i = 0; i < kMaxCuts; ++i) v[i] = i < p.cuts ? stats[first + i * kRows] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < PER; ++i)   // (what a part without keys has not written has no weight)
    y[i] = *reinterpret_cast<const float4*>(p.part + (first + min(i * G + g, p.cuts - 1) * kRows) * D + 4 * x);
  float top = -INFINITY, l = 0.0f, exact = 0.0f, seen = 0.0f;
#pragma unroll
  for (int i = 0; i < kMaxCuts; ++i) {
    if (v[i].y != 0.0f) top = fmaxf(top, v[i].x);
    seen = fmaxf(seen, v[i].w);
  }
#pragma unroll
  for (int i = 0; i < kMaxCuts; ++i) {
    v[i].x = v[i].y != 0.0f ? __builtin_amdgcn_exp2f(v[i].x - top) : 0.0f;
    l += v[i].x * v[i].y;
    exact += v[i].x * v[i].z;
  }
  float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    float w = 0.0f;
#pragma unroll
    for (int j = 0; j < G; ++j) w = g == j ? v[i * G + j].x : w;
    if (w == 0.0f) continue;
    o[0] += w * y[i].x;
    o[1] += w * y[i].y;
    o[2] += w * y[i].z;
    o[3] += w * y[i].w;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    o[e] = add_partner(o[e]);
    if (LANES <= 16) {
      const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(o[e]), __float_as_uint(o[e]), false, false);
      o[e] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    if (LANES <= 8) o[e] += xor_partner<8>(o[e]);
  }
  if (g != 0) return;
  const float inv = l == 0.0f ? (seen != 0.0f ? NAN : 0.0f) : 1.0f / l;
  *reinterpret_cast<uint2*>(p.out + to * D + 4 * x) =
      make_uint2(Mfma<T>::pack(o[0] * inv, o[1] * inv), Mfma<T>::pack(o[2] * inv, o[3] * inv));
  if (p.lse && x == 0) p.lse[to] = l == 0.0f ? -INFINITY : kLn2 * (top + __builtin_amdgcn_logf(exact));
}

// How a call is laid over the GPU.
struct Plan {
  bool walk, few;   // all keys of a workgroup's rows; those of at most 32 rows
  int64_t seq_tiles, all_tiles;
  int places, shares, own, piece;
  int64_t whole, left;
  int cuts;
  int64_t parts;   // rows of partial results
  int64_t table;   // sequences that have a line behind them
  int64_t bytes(int dim) const { return parts * (dim + 4) * 4 + table * 8; }
};

Plan plan(int64_t n, int64_t q_rows, int64_t k_rows, int64_t prefix, int heads, int kv_heads) {
  const int group = heads / kv_heads;
  const int64_t cus = compute_units(), rows = n * q_rows * heads;   // of the output
  Plan pl = {};
  pl.seq_tiles = (q_rows * group + kRows - 1) / kRows;
  pl.all_tiles = (n * q_rows * group + kRows - 1) / kRows;
  const double tiles_p = (double)((prefix + kKeys - 1) / kKeys), tiles_k = (double)((k_rows + kKeys - 1) / kKeys);
  // Two workgroups per CU are resident: as many full rounds of them as leave pieces to choose
  // beside the one that each cache and each of the prefix's row tiles takes (one token of 64
  // sequences, 4096 shared keys, 512 own at most, 40 heads over 8: 42 us in two rounds, 94 in
  // one; of 16 over 131072 shared ones 145 in one, 159 in two).
  const int64_t least = pl.all_tiles + pl.seq_tiles * n, round = 2 * cus / kv_heads > 0 ? 2 * cus / kv_heads : 1;
  const int64_t places = (least * 7 / 5 + round - 1) / round * round;
  // The most pieces of the prefix, and the least tiles of one, by the cost of joining: 1 us per
  // tile of keys against 0.4 ns per row and piece.
  const double s = fmin(fmin(sqrt(tiles_p / (0.0004 * (double)rows)), (double)(places / pl.all_tiles)), kMaxPieces);
  pl.shares = s > 1.0 ? (int)s : 1;
  const double each = fmax(1.0, fmin(sqrt(tiles_k / (0.0003 * (double)rows)), tiles_k));
  pl.piece = (int)ceil(tiles_k / each);
  if (pl.piece < 1) pl.piece = 1;
  pl.places = n > kListed ? 0 : (int)places;
  pl.own = (int)(n > kListed ? n : places / pl.seq_tiles);
  pl.parts = (pl.shares * n + pl.own) * q_rows * heads;
  pl.table = n + 1;
  // Either way in us: a tile of a row tile and head takes one, a part of a row 0.15 ns to join
  // (2 x 400 tokens behind 3000, 40 heads over 8: 79 us cut into pieces, walked 116 us).
  constexpr double kJoin = 0.00015;
  const double tiles = tiles_p + tiles_k;
  const double pieces = ((double)pl.all_tiles * tiles_p + (double)(n * pl.seq_tiles) * tiles_k) * kv_heads / (double)cus +
                        2.8 + (double)rows * (0.0006 + kJoin * pl.shares);
  // A walk: two workgroups per CU are resident, for which a tile takes twice as long as for one.
  // What is left behind full rounds is cut so that it fills the GPU once more, for a part
  // of a round (at most eight, for what is written and read again).
  const int64_t items = n * pl.seq_tiles * kv_heads, slots = 2 * cus, left = items % slots;
  const int64_t cuts = left > 0 ? slots / left : 1;
  pl.cuts = cuts > kMaxCuts ? kMaxCuts : (int)cuts;
  double walk = (double)(items / slots) * tiles * 2.0;
  if (pl.cuts > 1) walk += ceil(tiles / pl.cuts) * 2.0 + 2.8 + (double)(left * kRows) * (0.0002 + kJoin * pl.cuts);
  else if (left > 0) walk += tiles * (left > cus ? 2.0 : 1.0);
  // At most 32 rows take their keys in half a tile's time and nothing is joined, for the cost of a
  // kernel less, 10 us with its launch, and 3 more for every round of pieces past two (one token
  // of 32 sequences over 1024 own keys at most, 40 heads over 8: 16.5 us, 23.4 in pieces; of 57
  // behind 164 shared and 157 own ones, 56 heads: 11.1 and 22.5; four of 39 behind 216, 56 key heads:
  // 39 and 51; one of 64 behind 4096, 40 heads: 66 and 35).
  pl.few = q_rows * group <= 32;
  if (pl.few) {
    const int64_t grid = (pl.places ? pl.places : pl.shares * pl.all_tiles + n * pl.seq_tiles) * kv_heads;
    const double rounds = ceil((double)grid / (double)slots);
    walk = ceil((double)items / (double)slots) * (tiles * (items <= cus ? 0.55 : 0.85) + 3.5) + 1.0 - 10.0 -
           3.0 * fmax(0.0, rounds - 2.0);
  }
  pl.walk = walk <= pieces || rows > kMaxBlocks;
  if (pl.walk && pl.few) {
    pl.parts = pl.table = 0;
  } else if (pl.walk) {
    pl.left = pl.cuts > 1 ? left : 0;
    pl.whole = items - pl.left;
    pl.parts = pl.left * pl.cuts * kRows;
    pl.table = 0;
  }
  return pl;
}

template <typename T, int D>
int launch(const PrefixArgs& p, const Plan& pl, hipStream_t s) {
  if (pl.walk && pl.few) {
    const int64_t grid = (int64_t)p.n * p.kv_heads;
    LR_REQUIRE(grid <= kMaxBlocks, "attention_prefix: %lld workgroups are not supported", (long long)grid);
    prefix_walk_few<T, D><<<(unsigned)grid, 256, 0, s>>>(p);
    return check_launch("attention_prefix");
  }
  if (pl.walk) {
    const int64_t grid = pl.whole + pl.left * pl.cuts;
    LR_REQUIRE(grid <= kMaxBlocks, "attention_prefix: %lld workgroups are not supported", (long long)grid);
    if (p.lse) prefix_walk<T, D, true><<<(unsigned)grid, 256, 0, s>>>(p);
    else prefix_walk<T, D, false><<<(unsigned)grid, 256, 0, s>>>(p);
    if (int rc = check_launch("attention_prefix")) return rc;
    if (pl.left == 0) return LR_OK;
    walk_join<T, D><<<(unsigned)(pl.left * kRows / 4), 256, 0, s>>>(p);
    return check_launch("attention_prefix");
  }
  const int64_t grid = (p.places ? p.places : pl.shares * pl.all_tiles + p.n * pl.seq_tiles) * p.kv_heads;
  LR_REQUIRE(grid <= kMaxBlocks, "attention_prefix: %lld workgroups are not supported", (long long)grid);
  prefix_pieces<T, D><<<(unsigned)grid, 256, 0, s>>>(p);
  if (int rc = check_launch("attention_prefix")) return rc;
  prefix_join<T, D><<<(unsigned)((int64_t)p.n * p.q_rows * p.heads), 256, 0, s>>>(p);
  return check_launch("attention_prefix");
}

template <typename T>
int by_dim(const PrefixArgs& p, int dim, const Plan& pl, hipStream_t s) {
  if (dim == 32) return launch<T, 32>(p, pl, s);
  if (dim == 64) return launch<T, 64>(p, pl, s);
  return launch<T, 128>(p, pl, s);
}

int check_shape(int64_t n, int64_t q_rows, int64_t k_rows, int64_t prefix, int heads, int kv_heads, int head_dim) {
  LR_REQUIRE(n >= 0 && q_rows >= 0 && k_rows >= 0 && prefix >= 0, "attention_prefix: negative shape");
  LR_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0,
             "attention_prefix: %d heads do not share %d key heads evenly", heads, kv_heads);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(LR_EUNSUPPORTED, "attention_prefix: head_dim %d is not supported (32, 64 or 128)", head_dim);
  LR_REQUIRE(n < (1LL << 24) && q_rows < (1LL << 30) && k_rows < (1LL << 30) && prefix < (1LL << 30) && heads <= 65536,
             "attention_prefix: shapes past 2^24 sequences, 2^30 rows or 65536 heads are not supported");
  LR_REQUIRE(q_rows == 0 || n < (1LL << 30) / q_rows / heads, "attention_prefix: %lld x %lld tokens of %d heads are not supported",
             (long long)n, (long long)q_rows, heads);
  return LR_OK;
}

}  // namespace
}  // namespace lr

using namespace lr;

extern "C" int lr_attention_prefix_workspace(int64_t sequences, int64_t q_rows, int64_t k_rows, int64_t prefix_rows,
                                             int heads, int kv_heads, int head_dim, int64_t* bytes) {
  if (int rc = check_shape(sequences, q_rows, k_rows, prefix_rows, heads, kv_heads, head_dim)) return rc;
  LR_REQUIRE(bytes, "attention_prefix: null pointer");
  *bytes = 0;
  if (sequences == 0 || q_rows == 0) return LR_OK;
  const Plan pl = plan(sequences, q_rows, k_rows, prefix_rows, heads, kv_heads);
  *bytes = pl.bytes(head_dim);
  return LR_OK;
}

extern "C" int lr_attention_prefix(const void* q, const void* prefix_k, const void* prefix_v, const void* k, const void* v,
                                   void* out, float* lse, int dtype, int64_t sequences, int64_t q_rows, int64_t k_rows,
                                   int64_t prefix_rows, int heads, int kv_heads, int head_dim, const int64_t* strides,
                                   const int32_t* key_lengths, int causal, int scale_bits, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  LR_REQUIRE(dtype == LR_DTYPE_BF16 || dtype == LR_DTYPE_F16, "attention_prefix: unknown dtype %d", dtype);
  if (int rc = check_shape(sequences, q_rows, k_rows, prefix_rows, heads, kv_heads, head_dim)) return rc;
  if (sequences == 0 || q_rows == 0) return LR_OK;
  LR_REQUIRE(q && out && strides && (k_rows == 0 || (k && v)) && (prefix_rows == 0 || (prefix_k && prefix_v)),
             "attention_prefix: null pointer");
  LR_REQUIRE(aligned(q, 16) && aligned(prefix_k, 16) && aligned(prefix_v, 16) && aligned(k, 16) && aligned(v, 16) &&
                 aligned(out, 16) && aligned(lse, 4),
             "attention_prefix: pointers must be 16-byte aligned");
  for (int i = 0; i < 13; ++i)
    LR_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0,
               "attention_prefix: stride %d is %lld, not a multiple of 8 from 0 on", i, (long long)strides[i]);
  // A tile's keys are addressed by 32-bit byte offsets from its first one.
  for (int i : {3, 5, 7, 10})
    LR_REQUIRE(strides[i] < (1LL << 23),
               "attention_prefix: strides of 2^23 and more between keys or values are not supported");
  PrefixArgs p = {};
  p.q = static_cast<const uint16_t*>(q);
  p.pk = static_cast<const uint16_t*>(prefix_k);
  p.pv = static_cast<const uint16_t*>(prefix_v);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.out = static_cast<uint16_t*>(out);
  p.lse = lse;
  p.part = static_cast<float*>(workspace);
  p.qt = strides[0]; p.qh = strides[1]; p.qb = strides[2];
  p.pkt = strides[3]; p.pkh = strides[4]; p.pvt = strides[5]; p.pvh = strides[6];
  p.kt = strides[7]; p.kh = strides[8]; p.kb = strides[9];
  p.vt = strides[10]; p.vh = strides[11]; p.vb = strides[12];
  p.lengths = key_lengths;
  p.n = (int)sequences;
  p.q_rows = (int)q_rows;
  p.k_rows = (int)k_rows;
  p.prefix = (int)prefix_rows;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = heads / kv_heads;
  p.causal = causal != 0;
  float scale;
  static_assert(sizeof scale == sizeof scale_bits, "fp32");
  __builtin_memcpy(&scale, &scale_bits, sizeof scale);
  p.c = scale * 1.4426950408889634f;
  LR_REQUIRE(p.c > 0.0f && isfinite(p.c), "attention_prefix: the scale must be positive and finite");
  const Plan pl = plan(sequences, q_rows, k_rows, prefix_rows, heads, kv_heads);
  p.seq_tiles = (int)pl.seq_tiles;
  p.all_tiles = (int)pl.all_tiles;
  p.places = pl.places;
  p.shares = pl.shares;
  p.own = pl.own;
  p.piece = pl.piece;
  p.whole = (int)pl.whole;
  p.left = (int)pl.left;
  p.cuts = pl.cuts;
  if (pl.bytes(head_dim))
    LR_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= pl.bytes(head_dim),
               "attention_prefix: needs a workspace of %lld bytes", (long long)pl.bytes(head_dim));
  hipStream_t s = as_stream(stream);
  return dtype == LR_DTYPE_BF16 ? by_dim<__bf16>(p, head_dim, pl, s) : by_dim<_Float16>(p, head_dim, pl, s);
}
