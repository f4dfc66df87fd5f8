// attention.hip - softmax(scale * Q K^T) V for bf16 and fp16, head_dim 32, 64, 128.
//
// One pass over the keys with a running maximum m and sum l per query row:
//   s = scale * q . k;  m' = max(m, s);  p = 2^(log2(e) (s - m'));
//   l = l 2^(log2(e) (m - m')) + sum p;  o = o 2^(log2(e) (m - m')) + p V
// and o / l at the end: 0 where a row sees no key, NaN where all that it sees score -inf
// (l is 0 in both). Scores, m, l and o are fp32; p is rounded to the inputs' type for
// the second product, and o / l once at the end.
// l adds the rounded p (in fp32, by a dot product with ones): the weights p / l then
// add up to one, and a rounding error of p counts with v - o instead of v. Few rows
// (FEW) leave the matrix units time to spare: there p is the sum of two such numbers.
//
// Both products run transposed on the 32x32x16 MFMA, S^T = K Q^T and O^T = V^T P^T:
// lane l then holds keys of query l % 32 only, so maxima and sums are over a
// lane's own registers and its partner l ^ 32, and the score registers of 16 keys
// are, converted and packed, the second product's operand: the contraction runs
// over the keys in whatever order both operands agree on, here key 4 * (l / 32) +
// j % 4 + 8 * (j / 4) for slot j. V^T comes out of row-major LDS by the
// transposing read (ds_read_b64_tr_b16), four keys of a column per lane.
//
// m is moved only when a tile's maximum exceeds it by more than 2^kSlack (any m
// gives the same quotient o / l; p stays below 2^kSlack): most tiles then skip
// the multiplication of o.
#include "lr_attention.h"
#include "lr_runtime.h"

namespace lr {
namespace {

struct AttnArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  float* part;           // split keys: o [splits][rows][dim], then (m, l) [splits][rows]
  int64_t qt, qh, qb;    // strides of a token, a head, a sequence, in elements
  int64_t kt, kh, kb;
  int64_t vt, vh, vb;
  const int32_t* cu_q;   // packed sequences: n + 1 first rows, else null
  const int32_t* cu_k;
  const int32_t* lengths;  // valid keys per sequence of a dense batch, or null
  int64_t n, q_rows, k_rows;  // sequences; rows per sequence (dense) or in all (packed)
  int heads, kv_heads, group;   // group = heads / kv_heads: query heads that share a key head and a tile's rows
  int causal, splits;
  float c;               // scale * log2(e)
  int tiles, seq_tiles;  // row tiles per head in all (pieces: of a sequence), and of a dense batch's sequence
  int piece;             // least keys of a piece
};

// A sequence's rows and keys. Values read from the device are clamped, so that
// wrong ones cannot lead outside the tensors.
struct Seq {
  int64_t q0, k0;  // first row / key (token index into q and k, before the batch stride)
  int64_t b;       // dense: sequence
  int qn, kn;
};


// Packed rows: sequence i = 0 stands for the rows before cu_q[0], n + 1 for those
// behind cu_q[n]; both have no keys.
__device__ __forceinline__ int64_t first_row(const AttnArgs& p, int64_t i) {
  return i == 0 ? 0 : (i == p.n + 2 ? p.q_rows : clamp64(p.cu_q[i - 1], 0, p.q_rows));
}

constexpr int kMaxSplits = 256;  // of a sequence

// Few queries over sequences of different numbers of keys: all are cut into pieces of
// one size, so that the longest is not what everybody waits for, in a list over the
// sequences that every wave works out from the lengths by itself. It has p.splits >= 2 n
// places for n sequences (lr_attention).
struct Pieces {
  int chunk = 0;              // keys of a piece, a multiple of 64
  int seq = -1, keys = 0;     // the sequence asked for (-1: the list ends before)
  int first = 0, count = 0;   // its pieces
  __device__ Pieces() {}
  // Of sequence `want`, or where that is -1 the one that has piece `place`.
  __device__ Pieces(const AttnArgs& p, int64_t want, int place) {
    const int lane = threadIdx.x & 63;
    auto length = [&](int64_t i) __attribute__((always_inline)) {
      return i < p.n ? (int)clamp64(p.lengths[i], 0, p.k_rows) : 0;
    };
    // The smallest pieces that the list holds: from an even share up in steps, which end
    // at the latest where n of the places are left for sequences' last pieces. Sums in
    // fp32, in units of 64 keys: they may pass 32 bits (sequences of an expanded tensor
    // share their keys); the counts that have to be exact are below 2^24.
    auto units_of = [&](int size) __attribute__((always_inline)) {
      float sum = 0.0f;
      for (int64_t i = lane; i < p.n; i += 64)
        sum += (float)((uint32_t)(((length(i) + 63) >> 6) + size - 1) / (uint32_t)size);
      // The same in every lane; said so, since what depends on it addresses memory.
      return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(wave_tree_sum(sum))));
    };
    const int least = (int)((p.k_rows + 64 * kMaxSplits - 1) / (64 * kMaxSplits));   // of one sequence
    const float share = units_of(1) / (float)p.splits;
    int size = max(max(p.piece >> 6, least), share < 1.6e7f ? (int)share : 1 << 24);
    while (units_of(size) > (float)p.splits) size += max(1, size >> 4);
    chunk = __builtin_amdgcn_readfirstlane(size) * 64;
    int before = 0;   // pieces of the sequences before this group of 64
    for (int64_t base = 0; base < p.n; base += 64) {
      const int mine = length(base + lane);
      const int n = (int)((uint32_t)(mine + chunk - 1) / (uint32_t)chunk);
      const int upto = wave_prefix_sum(n);   // pieces of this group's sequences up to the lane's
      const bool here = want >= 0 ? base + lane == want : (before + upto > place && base + lane < p.n);
      const uint64_t hit = __ballot(here);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        seq = (int)base + l;
        keys = __builtin_amdgcn_readlane(mine, l);
        count = __builtin_amdgcn_readlane(n, l);
        first = before + __builtin_amdgcn_readlane(upto, l) - count;
        return;
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
  }
};

// What a workgroup works on: its split, sequence, rows [r0, r0 + kRows) of the
// sequence's (row r: token r / group, head hd * group + r % group), and key tiles.
// All heads that share a key head share its tiles, so that keys are read once for them,
// a causal tile spans fewer tokens, and a few tokens leave less of it empty (eight packed
// prompts of 40 heads over 8: 253 us with tiles of one head each, 236 so; one token of
// them over 4096 keys: 27.0 and 13.0).
struct Item {
  Seq s;
  int rows, r0;
  int split, piece, hd;   // piece: over all sequences (Pieces); hd: key head
  int sure;     // keys that every row of the workgroup sees
  int t0, t1;   // its tiles of kKeys keys
};

// Everything fits 32 bits: workgroups are fewer than 2^24, rows than 2^31 (lr_attention).
__device__ __forceinline__ bool find_item(const AttnArgs& p, Item& it) {
  // Workgroups are dealt to the 8 XCDs in turn. Where all tiles cost the same, those of
  // a head lie together and each XCD takes a contiguous run, so that its L2 serves a
  // head's keys once. Where they do not (causal), the heads come first, so that
  // the largest tiles of every head start before the small ones of any (with eight
  // heads or a multiple an XCD then has heads of its own as well). Splits share no keys:
  // all heads of the same ones, which lie side by side, come first.
  const uint32_t total = gridDim.x, pid = blockIdx.x;
  int tile;
  if (p.splits > 1 || p.causal) {
    const uint32_t hds = (uint32_t)p.kv_heads, item = pid / hds;
    tile = (int)(item / (uint32_t)p.splits);
    it.hd = (int)(pid - item * hds);
    it.split = (int)(item - tile * p.splits);
  } else {
    const uint32_t per = total >> 3, rest = total & 7, xcd = pid & 7;
    const uint32_t lid = (xcd < rest ? xcd * (per + 1) : rest * (per + 1) + (xcd - rest) * per) + (pid >> 3);
    it.split = 0;
    it.hd = (int)(lid / (uint32_t)p.tiles);
    tile = (int)(lid - it.hd * p.tiles);
  }
  Seq s = {};
  int tiles;   // of the sequence
  Pieces pc = {};
  const bool ragged = p.lengths && p.splits > 1;
  if (ragged) {
    pc = Pieces(p, -1, it.split);
    if (pc.seq < 0) return false;
    it.piece = it.split;
    it.split -= pc.first;
    tiles = p.tiles;
    s.b = pc.seq;
    s.qn = (int)p.q_rows;
    s.kn = pc.keys;
  } else if (p.cu_q) {
    // Sequence i has the tile slots from first_row(i) * group / kRows + i on: at least
    // as many as its rows need, and its own.
    const int slot = tile;
    auto start = [&](int i) __attribute__((always_inline)) {
      return (int)((uint32_t)(first_row(p, i) * p.group) / kRows) + i;
    };
    // The last sequence whose first slot is not behind this one: the lanes probe 64
    // places at once, so that a thousand sequences cost two loads in turn.
    int lo = 0, hi = (int)p.n + 1;
    while (lo < hi) {
      const int step = (hi - lo + 64) >> 6, at = lo + (int)(threadIdx.x & 63) * step;
      const uint64_t hit = __ballot(at <= hi && start(at) <= slot);
      lo += (__builtin_popcountll(hit) - 1) * step;
      hi = min(hi, lo + step - 1);
    }
    s.q0 = first_row(p, lo);
    s.qn = (int)clamp64(first_row(p, lo + 1) - s.q0, 0, p.q_rows);
    tile = slot - start(lo);
    tiles = (int)((uint32_t)(s.qn * p.group + kRows - 1) / kRows);
    if (lo > 0 && lo <= p.n) {
      s.k0 = clamp64(p.cu_k[lo - 1], 0, p.k_rows);
      s.kn = (int)clamp64(clamp64(p.cu_k[lo], 0, p.k_rows) - s.k0, 0, p.k_rows);
    }
    // (A list that is not in order can end the search at a sequence behind this slot.)
    if (tile < 0 || tile >= tiles) return false;
  } else {
    tiles = p.seq_tiles;
    const int b = (int)((uint32_t)tile / (uint32_t)tiles);
    s.b = b;
    tile -= b * tiles;
    s.qn = (int)p.q_rows;
    s.kn = (int)(p.lengths ? clamp64(p.lengths[b], 0, p.k_rows) : p.k_rows);
  }
  // Causal: the last tiles see the most keys and go first.
  if (p.causal) tile = tiles - 1 - tile;
  it.s = s;
  it.rows = s.qn * p.group;
  it.r0 = tile * kRows;
  it.sure = s.kn;
  int seen = s.kn;
  if (p.causal) {
    const int last = min(it.r0 + kRows, it.rows) - 1;
    seen = min(s.kn, max(0, s.kn - s.qn + (int)((uint32_t)last / (uint32_t)p.group) + 1));
    it.sure = min(s.kn, max(0, s.kn - s.qn + (int)((uint32_t)it.r0 / (uint32_t)p.group) + 1));
  }
  const int tiles_k = (seen + kKeys - 1) / kKeys;
  const int chunk = ragged ? pc.chunk / kKeys : (tiles_k + p.splits - 1) / p.splits;
  it.t0 = min(tiles_k, it.split * chunk);
  it.t1 = min(tiles_k, it.t0 + chunk);
  return true;
}

// The query row of a lane (column `col` of a wave's 32 rows from `r` on).
struct QueryRow {
  int64_t off;   // of its first element in q
  int r, tok, head, limit;   // limit: keys that it sees
  __device__ __forceinline__ QueryRow(const AttnArgs& p, const Item& it, int row) : r(row) {
    const int rc = row < it.rows ? row : it.rows - 1;
    tok = (int)((uint32_t)rc / (uint32_t)p.group);
    head = it.hd * p.group + (rc - tok * p.group);
    off = it.s.b * p.qb + (it.s.q0 + tok) * p.qt + head * p.qh;
    limit = p.causal ? min(it.s.kn, max(0, it.s.kn - it.s.qn + tok + 1)) : it.s.kn;
  }
};

// o / l, or a split's o, m and l; lane holds columns 32 * d + 8 * g + 4 * half + 0..3 of its row.
template <typename T, int D>
__device__ __forceinline__ void store_row(const AttnArgs& p, const Item& it, const QueryRow& qr, float m, float l,
                                          const v16f (&o)[D / 32], int half) {
  const float sum = add_partner(l);
  if (qr.r >= it.rows) return;
  const int64_t row = (it.s.b * p.q_rows + it.s.q0 + qr.tok) * p.heads + qr.head;
  if (p.splits > 1) {
    const int64_t all = (p.cu_q || p.lengths ? 1 : p.n) * p.q_rows * p.heads;   // rows of a split
    const int64_t at = p.lengths ? it.piece * all + (int64_t)qr.tok * p.heads + qr.head : it.split * all + row;
    float* const po = p.part + at * D;
    float* const ml = p.part + (int64_t)p.splits * all * D + at * 2;
    if (half == 0) {
      // Without a sum: whether the row has keys here (m is -inf either way).
      ml[0] = sum == 0.0f && qr.limit > it.t0 * kKeys ? INFINITY : m;
      ml[1] = sum;
    }
    if (sum == 0.0f) return;   // left out of the join by its l
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(po + 32 * d + 8 * g + 4 * half) =
            make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
    return;
  }
  const float inv = sum == 0.0f ? (qr.limit > 0 ? NAN : 0.0f) : 1.0f / sum;
  uint16_t* const po = p.out + row * D;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<uint2*>(po + 32 * d + 8 * g + 4 * half) =
          make_uint2(Mfma<T>::pack(o[d][4 * g] * inv, o[d][4 * g + 1] * inv),
                     Mfma<T>::pack(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv));
}

// -------------------------------------------------------------- kernel ----
// Few rows (FEW) or the pipeline, see lr_attention.h.
template <typename T, int D, bool FEW>
__global__ __launch_bounds__(256, 2) void attention(AttnArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[kTileBytes<D>];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  Item it;
  if (!find_item(p, it)) return;
  const Seq s = it.s;
  const QueryRow qr(p, it, it.r0 + wave * 32 + (lane & 31));
  const OneCache keys = {p.k + s.b * p.kb + s.k0 * p.kt + it.hd * p.kh, p.v + s.b * p.vb + s.k0 * p.vt + it.hd * p.vh,
                         p.kt, p.vt, s.kn, it.sure, qr.limit};
  v16f o[D / 32];
  float m, l, exact, off;
  attend<T, D, FEW, false>(smem, keys, p.q + qr.off, p.c, it.t0, it.t1, it.r0 + wave * 32 >= it.rows, m, l, exact, off,
                           o);
  store_row<T, D>(p, it, qr, m, l, o, lane >> 5);
}

// Joins the splits of a row: weights 2^(c (m_s - max m)). A workgroup per row: D / 4
// threads hold a split's columns, and the groups of them take every G-th split,
// then are added in order, so that the result does not depend on timing.
template <typename T, int D>
__global__ __launch_bounds__(256) void join_splits(AttnArgs p) {
  constexpr int LANES = D / 4, G = 256 / LANES;
  __shared__ float weight[256];
  __shared__ float4 sums[G][LANES];
  const int64_t row = blockIdx.x;
  const int64_t rows = (p.cu_q || p.lengths ? 1 : p.n) * p.q_rows * p.heads;   // of a split
  const float* const part = p.part;
  const float2* const ml = reinterpret_cast<const float2*>(part + (int64_t)p.splits * rows * D);
  // The row of its first split, and how many it has.
  int64_t at0 = row;
  int splits = p.splits;
  if (p.lengths) {
    const int64_t seq = row / rows;
    const Pieces pc(p, seq, 0);
    at0 = pc.first * rows + (row - seq * rows);
    splits = pc.count;
  }
  const int t = threadIdx.x, at = t % LANES, g = t / LANES;
  // Every wave finds the maximum and the sum by itself (at most 256 splits).
  float2 v[4];
  float m = -INFINITY;
  bool keys = false;   // whether a split without a sum has some of the row (store_row)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int s = 64 * i + (t & 63);
    v[i] = s < splits ? ml[at0 + s * rows] : make_float2(0.0f, 0.0f);
    if (v[i].y != 0.0f) m = fmaxf(m, v[i].x);
    else keys |= v[i].x == INFINITY;
  }
  m = wave_max(m);
  float l = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float w = v[i].y != 0.0f ? __builtin_amdgcn_exp2f((v[i].x - m) * p.c) : 0.0f;
    weight[64 * i + (t & 63)] = w;   // the same value from each wave
    l += w * v[i].y;
  }
  l = wave_tree_sum(l);
  const bool sees = __any(keys);
  __syncthreads();
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  constexpr int BATCH = 4;   // loads in flight
  for (int s0 = g; s0 < splits; s0 += BATCH * G) {
    float4 x[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (s0 + i * G < splits) x[i] = *reinterpret_cast<const float4*>(part + (at0 + (s0 + i * G) * rows) * D + 4 * at);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const float w = s0 + i * G < splits ? weight[s0 + i * G] : 0.0f;
      if (w == 0.0f) continue;   // x was not written where the split had no keys
      o.x += w * x[i].x;
      o.y += w * x[i].y;
      o.z += w * x[i].z;
      o.w += w * x[i].w;
    }
  }
  sums[g][at] = o;
  __syncthreads();
  if (g != 0) return;
#pragma unroll
  for (int i = 1; i < G; ++i) {
    const float4 x = sums[i][at];
    o.x += x.x;
    o.y += x.y;
    o.z += x.z;
    o.w += x.w;
  }
  const float inv = l == 0.0f ? (sees ? NAN : 0.0f) : 1.0f / l;
  *reinterpret_cast<uint2*>(p.out + row * D + 4 * at) =
      make_uint2(Mfma<T>::pack(o.x * inv, o.y * inv), Mfma<T>::pack(o.z * inv, o.w * inv));
}

// How a call is laid over the GPU.
struct Plan {
  int piece, splits;     // least keys of a piece; splits of the keys
  int64_t tiles;         // row tiles per key head in all (pieces: of a sequence)
  bool few;              // one wave's rows
  bool pieces = false;   // splits counts pieces of all sequences
};

Plan plan(int64_t n, int64_t q_rows, int64_t k_rows, int kind, int heads, int kv_heads) {
  const bool packed = kind == LR_ATTN_PACKED;
  const int group = heads / kv_heads;
  const int64_t mean_q = packed ? (n > 0 ? q_rows / n : 0) : q_rows;   // rows per sequence
  const int64_t mean_k = packed ? (n > 0 ? k_rows / n : 0) : k_rows;
  Plan pl;
  pl.tiles = packed ? q_rows * group / kRows + n + 2 : n * ((q_rows * group + kRows - 1) / kRows);
  const int64_t work = pl.tiles * kv_heads;
  const int64_t tile_rows = mean_q * group < kRows ? mean_q * group : kRows;
  // Workgroups to aim at. One wave's rows: two per CU, for the stream of keys (one token,
  // 32768 keys, 8 heads of 64: 16.9 us, 19.8 with one). Several waves': one per CU, since
  // two share its matrix units and leave twice the partial results (300 tokens, 4096
  // keys, 8 heads: 20.0 us with 8 splits, 22.5 with 12).
  const int64_t want = (tile_rows <= 32 ? 2 : 1) * compute_units();
  // (Packed rows have one kernel whatever lies around a sequence: the same bits.)
  pl.few = tile_rows <= 32 && !packed;
  // A split takes 1 us per tile of keys; joining s of them 2.8 us, and per row 0.6 ns and
  // 0.15 ns per split (head_dim 128, from 12 shapes). So the best s is the root of
  // tiles / (0.00015 rows), and one where joining costs more than it saves: 878 tokens,
  // 8 heads, take 19.6 us as they are and 20.6 with 4 splits; 128 tokens, 40 heads, 4096
  // keys 77.8 and 31.9 with 6. Two tiles per split at least (one token, 4096 keys, 8 heads:
  // 11.2 us, 12.4 with one).
  const double tiles_k = (double)((mean_k + kKeys - 1) / kKeys), rows = (double)((packed ? 1 : n) * q_rows * heads);
  double s = sqrt(tiles_k / (0.00015 * rows));
  s = fmin(fmin(s, tiles_k / 2), work > 0 ? (double)(want / work) : 1.0);
  s = fmin(floor(s), kMaxSplits);
  if (s > 1.0 && tiles_k / s + 2.8 + rows * (0.0006 + 0.00015 * s) > tiles_k) s = 1.0;
  pl.splits = s > 1.0 ? (int)s : 1;
  pl.piece = kKeys;
  if (kind == LR_ATTN_LENGTHS && pl.splits > 1) {
    // Places of a list of pieces over all sequences: as many as fill the GPU (one
    // workgroup more would take a second round), at least 2 n, since want / work is 2 or
    // more here; past that (257 pairs of a sequence and a key head with few rows on 256
    // CUs) every sequence is walked whole. Least keys of a piece by the same cost, halved
    // since the caches are rarely all full: 32 rows over three caches of 4096, 16 heads,
    // take 31.3 us with 512 keys and 35.7 with 64; 5 rows over four of 512 8.9 with 64 and
    // 9.7 with 128.
    const double each = fmin(sqrt(tiles_k / (0.0003 * rows)), tiles_k);
    pl.piece = (int)ceil((double)mean_k / fmax(each, 1.0) / kKeys) * kKeys;
    const int64_t most = mean_k / pl.piece;
    if (most < 2) {
      pl.splits = 1;
      return pl;
    }
    pl.pieces = true;
    pl.tiles /= n;
    const int64_t places = want / (pl.tiles * kv_heads);
    const int64_t all = n + n * (most < kMaxSplits ? most : kMaxSplits);
    pl.splits = (int)(places > all ? all : places);
  }
  return pl;
}

template <typename T, int D>
int launch(AttnArgs p, const Plan& pl, hipStream_t s) {
  const int64_t grid = pl.tiles * p.kv_heads * pl.splits;
  LR_REQUIRE(grid <= kMaxBlocks, "attention: %lld workgroups are not supported", (long long)grid);
  const int64_t rows = (p.cu_q ? 1 : p.n) * p.q_rows * p.heads;   // of the output
  LR_REQUIRE(pl.splits == 1 || rows <= kMaxBlocks, "attention: %lld rows are not supported with split keys",
             (long long)rows);
  if (pl.few) attention<T, D, true><<<(unsigned)grid, 256, 0, s>>>(p);
  else attention<T, D, false><<<(unsigned)grid, 256, 0, s>>>(p);
  if (int rc = check_launch("attention")) return rc;
  if (pl.splits == 1) return LR_OK;
  join_splits<T, D><<<(unsigned)rows, 256, 0, s>>>(p);
  return check_launch("attention");
}

template <typename T>
int by_dim(const AttnArgs& p, int dim, const Plan& pl, hipStream_t s) {
  if (dim == 32) return launch<T, 32>(p, pl, s);
  if (dim == 64) return launch<T, 64>(p, pl, s);
  return launch<T, 128>(p, pl, s);
}

}  // namespace
}  // namespace lr

using namespace lr;

extern "C" int lr_attention_splits(int64_t sequences, int64_t q_rows, int64_t k_rows, int kind, int heads,
                                   int kv_heads) {
  if (sequences <= 0 || q_rows <= 0 || k_rows <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return 1;
  return plan(sequences, q_rows, k_rows, kind, heads, kv_heads).splits;
}

extern "C" int lr_attention(const void* q, const void* k, const void* v, void* out, int dtype, int64_t sequences,
                            int64_t q_rows, int64_t k_rows, int heads, int kv_heads, int head_dim, const int64_t* strides,
                            const int32_t* cu_q, const int32_t* cu_k, const int32_t* key_lengths, int causal,
                            int scale_bits, void* workspace, int64_t workspace_bytes, int splits, void* stream) {
  LR_REQUIRE(dtype == LR_DTYPE_BF16 || dtype == LR_DTYPE_F16, "attention: unknown dtype %d", dtype);
  LR_REQUIRE(sequences >= 0 && q_rows >= 0 && k_rows >= 0, "attention: negative shape");
  LR_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0,
             "attention: %d heads do not share %d key heads evenly", heads, kv_heads);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(LR_EUNSUPPORTED, "attention: head_dim %d is not supported (32, 64 or 128)", head_dim);
  LR_REQUIRE(!cu_q == !cu_k && !(cu_q && key_lengths),
             "attention: packed sequences need both lists of first rows and no key lengths");
  const bool packed = cu_q != nullptr;
  if (q_rows == 0 || (!packed && sequences == 0)) return LR_OK;
  LR_REQUIRE(q_rows < (1LL << 30) && k_rows < (1LL << 30) && sequences < (1LL << 30) && heads <= 65536,
             "attention: shapes past 2^30 rows or 65536 heads are not supported");
  LR_REQUIRE(q_rows * (heads / kv_heads) < (1LL << 31) - kRows, "attention: %lld rows of a key head are not supported",
             (long long)(q_rows * (heads / kv_heads)));
  LR_REQUIRE(q && out && (k_rows == 0 || (k && v)), "attention: null pointer");
  LR_REQUIRE(strides, "attention: null pointer");
  LR_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16),
             "attention: pointers must be 16-byte aligned");
  for (int i = 0; i < 9; ++i)
    LR_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0, "attention: stride %d is %lld, not a multiple of 8 from 0 on",
               i, (long long)strides[i]);
  // A tile's keys are addressed by 32-bit byte offsets from its first one.
  LR_REQUIRE(strides[3] < (1LL << 23) && strides[6] < (1LL << 23),
             "attention: strides of 2^23 and more between keys or values are not supported");
  AttnArgs p = {};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.out = static_cast<uint16_t*>(out);
  p.part = static_cast<float*>(workspace);
  p.qt = strides[0]; p.qh = strides[1]; p.qb = strides[2];
  p.kt = strides[3]; p.kh = strides[4]; p.kb = strides[5];
  p.vt = strides[6]; p.vh = strides[7]; p.vb = strides[8];
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.lengths = key_lengths;
  p.n = sequences;
  p.q_rows = q_rows;
  p.k_rows = k_rows;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = heads / kv_heads;
  p.causal = causal != 0;
  float scale;
  static_assert(sizeof scale == sizeof scale_bits, "fp32");
  __builtin_memcpy(&scale, &scale_bits, sizeof scale);
  p.c = scale * 1.4426950408889634f;
  LR_REQUIRE(p.c > 0.0f && isfinite(p.c), "attention: the scale must be positive and finite");
  Plan pl = plan(sequences, q_rows, k_rows, packed ? LR_ATTN_PACKED : (key_lengths ? LR_ATTN_LENGTHS : LR_ATTN_DENSE),
                 heads, kv_heads);
  LR_REQUIRE(splits >= 1 && (splits == 1 || splits <= (pl.splits > kMaxSplits ? pl.splits : kMaxSplits)),
             "attention: %d splits", splits);
  if (key_lengths && splits > 1)
    LR_REQUIRE(pl.pieces && splits == pl.splits && splits >= 2 * sequences,
               "attention: with key lengths, 1 or the %d splits of lr_attention_splits", pl.splits);
  else if (pl.pieces)   // one split: whole sequences
    pl.tiles *= sequences;
  pl.splits = splits;
  LR_REQUIRE(pl.tiles < (1LL << 31), "attention: %lld row tiles are not supported", (long long)pl.tiles);
  p.tiles = (int)pl.tiles;
  p.seq_tiles = packed || (key_lengths && splits > 1) ? 0 : (int)(pl.tiles / sequences);
  p.piece = pl.piece;
  p.splits = splits;
  if (splits > 1) {
    const int64_t rows = (packed || key_lengths ? 1 : sequences) * q_rows * heads;
    LR_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= splits * rows * (head_dim + 2) * 4,
               "attention: %d splits need a workspace of %lld bytes", splits,
               (long long)(splits * rows * (head_dim + 2) * 4));
  }
  hipStream_t s = as_stream(stream);
  return dtype == LR_DTYPE_BF16 ? by_dim<__bf16>(p, head_dim, pl, s) : by_dim<_Float16>(p, head_dim, pl, s);
}
