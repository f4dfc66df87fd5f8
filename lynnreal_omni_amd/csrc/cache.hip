// cache.hip - caches of bounded size: the attention weight that each key gets, and the
// choice of the keys that stay.
//
// Weights. With the logarithm of each row's softmax sum given, a key j of key head h gets
//   w[j] += sum over rows r of h that see j of exp(scale q_r . k_j - lse_r),
// rows being tokens x the query heads that share h. A sum over rows per key is the
// transpose of what attention does, so a workgroup keeps keys, in registers, and the
// queries go by: S^T = K Q^T on the 32x32x16 MFMA leaves a lane with 16 keys of one query,
// each added to its own fp32 sum; the sums over the 32 lanes come once at the end. Every
// key is read once, and the order of additions does not depend on timing. With few rows the keys'
// stream bounds it; with many the exponentials and the matrix instructions do (a prompt of 3683
// tokens, 40 heads over 8: 105 us causal, 157 where every row sees every key).
//
// Eviction reads the weights, finds for every cache and head the keys that stay, and moves
// their rows to another cache, in their order.
#include "lr_attention.h"
#include "lr_pieces.h"
#include "lr_runtime.h"

namespace lr {
namespace {

// x / d for x below 2^31 by a multiplication: with 2^(l - 1) < d <= 2^l and m = ceil(2^(31 + l) / d),
// m d exceeds 2^(31 + l) by less than d <= 2^l, which x < 2^31 cannot bring to the next quotient.
struct Divisor {
  uint32_t m;
  int shift;
  explicit Divisor(uint32_t d) {
    int l = 0;
    while ((1u << l) < d) ++l;
    shift = 31 + l;
    m = (uint32_t)(((1ULL << shift) + d - 1) / d);
  }
  __device__ __forceinline__ int of(int x) const { return (int)(((uint64_t)(uint32_t)x * m) >> shift); }
};

struct WeighArgs {
  const uint16_t *q, *k;
  const float *lse, *w;   // lse [n][q_rows][heads]; w, out [n][kv_heads][k_rows]
  float* out;
  float* part;            // sums of a share's first and last keys [kv_heads][shares][2][256]
  int64_t qt, qh, qb, kt, kh, kb;
  const int32_t* lengths;
  int n, q_rows, k_rows, heads, kv_heads, group;
  int causal;
  int shares;             // of a key head's work; 0: a workgroup for every 128 keys
  int places;             // few rows: pieces of all caches for a key head
  float c;                // scale * log2(e)
  float one_by_group;
  Divisor by_group;
};

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t rsrc, void* lds, uint32_t voffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)lds, 4, voffset, 0, 0, 0);
}

// Sum over the 32 lanes of a half of the wave.
__device__ __forceinline__ float half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  v += xor_partner<8>(v);
  v += xor_partner<4>(v);
  v += xor_partner<2>(v);
  return v + xor_partner<1>(v);
}

constexpr int kGroup = 128;        // keys
constexpr int kDealt = 256;        // keys of a group that is dealt out
constexpr int kShared = 64;        // caches at most that are dealt out in shares: one per lane
constexpr int kLeastShare = 256;   // rows

// A cache's keys in groups of KEYS, each with the rows that see any of it: from `first` on.
template <int KEYS>
struct Seen {
  int kn, rows, hidden, group, causal;   // causal: token t sees keys up to hidden + t
  __device__ __forceinline__ Seen(const WeighArgs& p, int seq)
      : kn(keys_of(p.lengths, seq, p.k_rows)), rows(p.q_rows * p.group), hidden(kn - p.q_rows), group(p.group), causal(p.causal) {}
  __device__ __forceinline__ int groups() const { return ceil_div(kn, KEYS); }
  __device__ __forceinline__ int first(int g) const { return causal ? max(0, g * KEYS - hidden) * group : 0; }   // < rows
  // The rows of groups 0 .. g - 1, one group's behind the other's. `whole` of them have all rows.
  __device__ __forceinline__ int64_t before(int g) const {
    const int whole = causal ? (hidden < 0 ? 0 : min(g, hidden / KEYS + 1)) : g;
    const int64_t m = g - whole;
    return (int64_t)g * rows - group * (m * (whole * KEYS - hidden) + KEYS / 2 * m * (m - 1));
  }
  // The group that has row x of them.
  __device__ __forceinline__ int find(int64_t x) const {
    int lo = 0, hi = groups() - 1;
    while (lo < hi) {
      const int mid = lo + (hi - lo + 1) / 2;
      if (before(mid) <= x) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }
};

// All caches' rows, one cache's behind the other's, dealt out in even shares. Every wave works it
// out from the lengths by itself.
struct Deal {
  int64_t upto;   // the caches 0 .. lane
  int64_t all, each;
  static __device__ __forceinline__ int64_t of_lane(int64_t v, int lane) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
                     (uint32_t)__builtin_amdgcn_readlane((int)v, lane));
  }
  __device__ __forceinline__ explicit Deal(const WeighArgs& p) {
    const int lane = threadIdx.x & 63;
    const Seen<kDealt> mine(p, min(lane, p.n - 1));
    upto = lane < p.n ? mine.before(mine.groups()) : 0;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int64_t y = __shfl_up(upto, o);
      upto += lane >= o ? y : 0;
    }
    all = of_lane(upto, 63);
    each = ((all + p.shares - 1) / p.shares + kKeys - 1) / kKeys * kKeys;
    each = of_lane(each < kLeastShare ? kLeastShare : each, 0);   // (a division is a vector's work)
  }
  __device__ __forceinline__ explicit Deal(int64_t known) : upto(known), all(0), each(0) {}
  __device__ __forceinline__ int cache_of(int64_t x) const { return __builtin_ctzll(__ballot(upto > x)); }
  __device__ __forceinline__ int64_t before(int seq) const { return seq ? of_lane(upto, seq - 1) : 0; }
};

// Four waves with KB blocks of 32 keys each; queries in tiles of 64 rows, with their sums,
// through a ring in the LDS that first holds the keys on their way to the registers. Swizzle as in
// lr_attention.h. KB = 1: a workgroup for every 128 keys. KB = 2, which halves what the
// queries' fragments take of the LDS: a workgroup has a share of its key head's work, rows of one
// group of keys after the other, and sums of a group that is not its alone go to `part`. (Equal
// runs of each group's rows instead left a third of the CUs idle where causal: the prompt of
// 3683 tokens 138 us. Tokens and heads of a tile's rows by whole divisions in every tile: 8% more.)
template <typename T, int D, int KB>
__global__ __launch_bounds__(256, 4 / KB) void weigh_keys(WeighArgs p) {
  typedef typename Mfma<T>::V V8;
  constexpr int ROW = 2 * D, CH = ROW / 16, RPB = 256 / ROW, PAIRS = ROW / 32, KD = D / 16;
  constexpr int WAVES = 4, TILE = kKeys * ROW, DMAS = TILE / 1024 / WAVES, KEYS = 128 * KB;
  constexpr bool DEALT = KB == 2;
  constexpr int RING = KEYS / kKeys, LOADS = DMAS + 1;   // slots that fit into the keys' LDS; DMAs per wave and tile
  // (One array for all of it: between two the compiler waits for every DMA before any read.)
  __shared__ __attribute__((aligned(1024))) char smem[KEYS * (ROW + 4) + RING * WAVES * kKeys * 4 + (DEALT ? kShared * 8 : 0)];
  float* const sums = reinterpret_cast<float*>(smem + KEYS * ROW);
  char* const lses = smem + KEYS * (ROW + 4);   // [RING][WAVES][64], each wave's own
  int64_t* const uptos = reinterpret_cast<int64_t*>(lses + RING * WAVES * kKeys * 4);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Heads, which lie side by side, first.
  const int share = (int)(blockIdx.x / (uint32_t)p.kv_heads), hd = (int)(blockIdx.x - share * p.kv_heads);
  // Adds rows r_from .. rows - 1 to group g's sums, which are then in `sums`.
  auto weigh = [&](int seq, int g, int r_from, int rows) __attribute__((always_inline)) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));   // what follows from it does not stay in registers between groups
    const int half = lane >> 5, col = lane & 31;
    const int kn = keys_of(p.lengths, seq, p.k_rows), hidden = kn - p.q_rows;
    const int key0 = g * KEYS, tiles = (rows - r_from + kKeys - 1) / kKeys;
    float acc[KB][16];
#pragma unroll
    for (int y = 0; y < KB; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[y][e] = 0.0f;
    auto publish = [&](auto left) __attribute__((always_inline)) {   // loads that may still be on their way
      constexpr int N = decltype(left)::value;
      __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x70 | 0xf00);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    // The 16-byte slots of a tile that this lane fetches: row and chunk.
    auto slot_row = [&](int i) __attribute__((always_inline)) { return ((wave * DMAS + i) * 64 + lane) / CH; };
    auto slot_chunk = [&](int i) __attribute__((always_inline)) {
      return ((wave * DMAS + i) * 64 + lane) % CH ^ (slot_row(i) / RPB % PAIRS) * 2;
    };
    const uint16_t* const kbase = p.k + seq * p.kb + hd * p.kh;
#pragma unroll
    for (int x = 0; x < KEYS / kKeys; ++x) {
      const int left = min(kKeys, kn - key0 - x * kKeys);   // keys past the last read as zero
      const __amdgpu_buffer_rsrc_t r = row_rsrc(kbase + (left > 0 ? (key0 + (int64_t)x * kKeys) * p.kt : 0),
                                                left > 0 ? ((int64_t)(left - 1) * p.kt + D) * 2 : 0);
#pragma unroll
      for (int i = 0; i < DMAS; ++i)
        dma16(r, smem + x * TILE + (wave * DMAS + i) * 1024, (uint32_t)(slot_row(i) * p.kt * 2 + slot_chunk(i) * 16));
    }
    publish(std::integral_constant<int, 0>{});
    V8 kf[KB][KD];
#pragma unroll
    for (int y = 0; y < KB; ++y) {
      const int row = (wave * KB + y) * 32 + col;
#pragma unroll
      for (int d = 0; d < KD; ++d)
        kf[y][d] = *reinterpret_cast<const V8*>(smem + row * ROW + ((2 * d + half) ^ (row / RPB % PAIRS) * 2) * 16);
    }
    __syncthreads();   // the keys are in registers: the queries may take their place
    const uint16_t* const qbase = p.q + seq * p.qb + (int64_t)hd * p.group * p.qh;
    const float* const lbase = p.lse + (int64_t)seq * p.q_rows * p.heads + hd * p.group;
    // The token, from r0's on, and the head that row r0 + i is of, where r0 is `ph` rows behind its
    // token's first: quotient and rest by `group` of a number below group + 64, in fp32 (its error
    // of 2^-17 at most is less than the half that keeps it from a whole number, 0.5 / group).
    auto token_of = [&](int i, int ph) __attribute__((always_inline)) { return (int)(((float)(ph + i) + 0.5f) * p.one_by_group); };
    uint32_t qoff[DMAS];   // as if of one token
#pragma unroll
    for (int i = 0; i < DMAS; ++i) qoff[i] = (uint32_t)(slot_row(i) * p.qh * 2 + slot_chunk(i) * 16);
    const uint32_t turn_q = (uint32_t)((p.qt - p.group * p.qh) * 2), turn_l = (uint32_t)(p.heads - p.group);
    // Rows past the last one, which are masked, read others between the first and the last, or
    // zero; tiles past the last one, which keep the count of loads the same, repeat that.
    auto issue = [&](int t) {
      const int slot = t % RING, r0 = r_from + min(t, tiles - 1) * kKeys, tok0 = p.by_group.of(r0), ph = r0 - tok0 * p.group;
      const int toks = min(kKeys, p.q_rows - tok0);   // that 64 rows from r0 on can have
      const __amdgpu_buffer_rsrc_t rs =
          row_rsrc(qbase + (int64_t)tok0 * p.qt, ((toks - 1) * p.qt + (p.group - 1) * p.qh + D) * 2);
      const uint32_t at = (uint32_t)(ph * p.qh * 2);
#pragma unroll
      for (int i = 0; i < DMAS; ++i)
        dma16(rs, smem + slot * TILE + (wave * DMAS + i) * 1024, qoff[i] + at + token_of(slot_row(i), ph) * turn_q);
      const __amdgpu_buffer_rsrc_t ls =
          row_rsrc(lbase + (int64_t)tok0 * p.heads, ((int64_t)(toks - 1) * p.heads + p.group) * 4);
      dma4(ls, lses + (slot * WAVES + wave) * kKeys * 4, (ph + lane + token_of(lane, ph) * turn_l) * 4);
    };
    float l2 = INFINITY;   // of the block before: its row's lse * log2(e)
    auto add = [&](const v16f (&s)[KB], int i, bool sees) __attribute__((always_inline)) {
      const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 16][i % 16], p.c, -l2));
      acc[i / 16][i % 16] += sees ? w : 0.0f;
    };
    // The scores of block b of a tile, while the exponentials of the block before run between the
    // matrix instructions.
    auto product = [&](v16f (&s)[KB], const char* qs, int b, const v16f (&before)[KB]) __attribute__((always_inline)) {
      constexpr int AHEAD = KD < 3 ? KD : 3;
      V8 qf[4];
      // (2 d + half) ^ turn, hidden so that its values for every d do not stay in registers.
      int turn = (half ^ (col / RPB % PAIRS) * 2) * 16;
      asm volatile("" : "+v"(turn));
      auto read = [&](int d) __attribute__((always_inline)) {
        return *reinterpret_cast<const V8*>(qs + (32 * b + col) * ROW + (turn ^ 32 * d));
      };
#pragma unroll
      for (int d = 0; d < AHEAD; ++d) qf[d] = read(d);
      const v16f zero = {};
#pragma unroll
      for (int d = 0; d < KD; ++d) {
        if (d + AHEAD < KD) qf[(d + AHEAD) & 3] = read(d + AHEAD);
#pragma unroll
        for (int y = 0; y < KB; ++y) s[y] = Mfma<T>::mul(kf[y][d], qf[d & 3], d ? s[y] : zero);
#pragma unroll
        for (int i = 16 * KB * d / KD; i < 16 * KB * (d + 1) / KD; ++i) {
          add(before, i, true);
          asm volatile("" : "+v"(acc[i / 16][i % 16]));   // here, not behind the branch that follows
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    v16f s0[KB] = {}, s1[KB] = {};
    auto block = [&](v16f (&s)[KB], v16f (&before)[KB], const char* qs, int t, int b, float sum2) __attribute__((always_inline)) {
      product(s, qs, b, before);
      l2 = sum2;
      const int wave0 = key0 + wave * KB * 32, r0 = r_from + t * kKeys + 32 * b, tok0 = p.by_group.of(r0);
      if (r0 + 32 <= rows && (!p.causal || hidden + tok0 + 1 >= wave0 + 32 * KB)) return;
      // The keys that the lane's row sees, from the lane's first one on. A score of -infinity
      // stands for the others, or an infinite sum for all of them.
      const int own = wave0 + 4 * half;
      const int lim = r0 + col >= rows ? 0 : (p.causal ? hidden + tok0 + token_of(col, r0 - tok0 * p.group) + 1 : kn) - own;
      auto sees = [&](int i) __attribute__((always_inline)) { return 32 * (i / 16) + 8 * (i % 16 >> 2) + (i & 3) < lim; };
      if (__ballot(lim > 0 && !(l2 > -INFINITY)) == 0) {
#pragma unroll
        for (int i = 0; i < 16 * KB; ++i) s[i / 16][i % 16] = sees(i) ? s[i / 16][i % 16] : -INFINITY;
        if (lim <= 0) l2 = INFINITY;
        return;
      }
      // A row whose sum is -infinity (all of its scores are) or NaN: a score of -infinity would give
      // NaN there, so that what it does not see is left out by a choice.
#pragma unroll
      for (int i = 0; i < 16 * KB; ++i) {
        add(s, i, sees(i));
        s[i / 16][i % 16] = 0.0f;
      }
      l2 = INFINITY;
    };
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) issue(i);
#pragma unroll 1
    for (int t = 0; t < tiles; ++t) {
      publish(std::integral_constant<int, (RING - 2) * LOADS>{});   // tile t; every wave is done with tile t - 1
      issue(t + RING - 1);
      const int slot = t % RING;
      const char* const qs = smem + slot * TILE;
      // lse * log2(e) of the lane's row in each block.
      float now[2];
#pragma unroll
      for (int b = 0; b < 2; ++b)
        now[b] = reinterpret_cast<const float*>(lses)[(slot * WAVES + wave) * kKeys + 32 * b + col] * kLog2e;
      block(s0, s1, qs, t, 0, now[0]);
      if (r_from + t * kKeys + 32 >= rows) {   // the last tile, without a second block
#pragma unroll
        for (int i = 0; i < 16 * KB; ++i) s1[i / 16][i % 16] = s0[i / 16][i % 16];
        break;
      }
      block(s1, s0, qs, t, 1, now[1]);
    }
#pragma unroll
    for (int i = 0; i < 16 * KB; ++i) add(s1, i, true);
    __builtin_amdgcn_s_waitcnt(0x70 | 0xf00);   // the last DMAs have landed before the LDS goes to another
#pragma unroll
    for (int i = 0; i < 16 * KB; ++i) {
      const int y = i / 16, e = i % 16;
      const float v = half_sum(acc[y][e]);
      if (col == 0) sums[(wave * KB + y) * 32 + 8 * (e >> 2) + 4 * half + (e & 3)] = v;
    }
    __syncthreads();
  };
  const int i = (int)threadIdx.x;
  if constexpr (!DEALT) {
    const int seq = share % p.n, g = share / p.n, key = g * KEYS + i;
    const Seen<KEYS> seen(p, seq);
    const bool any = g < seen.groups() && seen.rows > 0;
    if (any) weigh(seq, g, seen.first(g), seen.rows);
    if (i >= KEYS || key >= p.k_rows) return;
    const int64_t at = ((int64_t)seq * p.kv_heads + hd) * p.k_rows + key;
    p.out[at] = any && key < seen.kn ? p.w[at] + sums[i] : p.w[at];   // places behind the keys stay as they were
  } else {
    const Deal deal(p);
    uptos[i & 63] = deal.upto;   // the same from every wave
    const int64_t begin = share * deal.each, end = min(deal.all, begin + deal.each);
    for (int64_t x = begin; x < end;) {
      const Deal known(uptos[i & 63]);
      const int seq = known.cache_of(x);
      const Seen<KEYS> seen(p, seq);
      const int64_t here = x - known.before(seq);
      const int g = __builtin_amdgcn_readfirstlane(seen.find(here)), key = g * KEYS + i, first = seen.first(g);
      const int r_from = first + (int)(here - seen.before(g)), to = (int)min((int64_t)seen.rows, r_from + (end - x));
      weigh(seq, g, r_from, to);
      if (key < keys_of(p.lengths, seq, p.k_rows)) {
        const int64_t at = ((int64_t)seq * p.kv_heads + hd) * p.k_rows + key;
        if (r_from == first && to == p.q_rows * p.group) p.out[at] = p.w[at] + sums[i];
        else p.part[(((int64_t)hd * p.shares + share) * 2 + (x != begin)) * KEYS + i] = sums[i];
      }
      x += to - r_from;
    }
  }
}

// Adds to the keys of a group that several shares have what each of them found, in order. Places
// behind the caches' keys stay as they were.
__global__ __launch_bounds__(kDealt) void join_shares(WeighArgs p) {
  const int hd = (int)(blockIdx.x % (uint32_t)p.kv_heads), rest = (int)(blockIdx.x / (uint32_t)p.kv_heads);
  const int seq = rest % p.n, g = rest / p.n, i = (int)threadIdx.x, key = g * kDealt + i;
  const Seen<kDealt> seen(p, seq);
  const Deal deal(p);
  if (key >= p.k_rows) return;
  const int64_t at = ((int64_t)seq * p.kv_heads + hd) * p.k_rows + key;
  if (key >= seen.kn || deal.all == 0) {
    if (p.out != p.w) p.out[at] = p.w[at];
    return;
  }
  const int64_t from = deal.before(seq) + seen.before(g), to = deal.before(seq) + seen.before(g + 1);
  const int s0 = (int)(from / deal.each), s1 = (int)((to - 1) / deal.each);
  if (s0 == s1) return;   // that share has written it
  float v = 0.0f;
  for (int s = s0; s <= s1; ++s) {
    // It is the first of a share's groups where the share begins inside of it.
    const float* const part = p.part + (((int64_t)hd * p.shares + s) * 2 + (s * deal.each < from)) * kDealt;
    v += part[i];
  }
  p.out[at] = p.w[at] + v;
}

// At most 32 rows per key head: what counts is the stream of keys. They are cut into pieces
// over all caches (lr_pieces.h); a wave has 32 keys of each 128 of them, through 32 rows of
// LDS of its own, and the queries in registers, so that no wave waits for another. The next
// keys are on their way while these are worked on.
// (Eight caches of 16152 keys in all, places for 65536, 40 heads over 8: 11-12 us; 17.2 with a
// workgroup for every 128 places of every cache. One of 131072 keys: 45 us, 6 TB/s, part of it out of the caches.)
constexpr int kCopied = 1024;   // places behind the caches' keys that a workgroup copies at a time

template <typename T, int D>
__global__ __launch_bounds__(256, 4) void weigh_few(WeighArgs p) {
  typedef typename Mfma<T>::V V8;
  constexpr int ROW = 2 * D, CH = ROW / 16, RPB = 256 / ROW, PAIRS = ROW / 32, KD = D / 16, DMAS = 32 * ROW / 1024;
  __shared__ __attribute__((aligned(1024))) char smem[4 * 32 * ROW];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int half = lane >> 5, col = lane & 31;
  const int place = (int)(blockIdx.x / (uint32_t)p.kv_heads), hd = (int)(blockIdx.x - place * p.kv_heads);
  Pieces caches;
  caches.load(p.lengths, p.n, p.k_rows, kGroup);
  // The smallest pieces that all have a place (there are n at least).
  int size = max(1, (int)(caches.count(1) / (float)p.places));
  while (caches.count(size) > (float)p.places) size += max(1, size >> 4);
  int seq, first = 0;
  caches.find(p.n, size, place, seq, first);
  if (seq >= 0) {
    const int kn = keys_of(p.lengths, seq, p.k_rows), hidden = kn - p.q_rows, all = ceil_div(kn, kGroup);
    const int each = Pieces::even(all, ceil_div(all, size));
    const int g0 = (place - first) * each, g1 = min(all, g0 + each);
    const uint16_t* const kbase = p.k + seq * p.kb + hd * p.kh;
    char* const mine = smem + wave * 32 * ROW;
    auto issue = [&](int g) {
      const int key = g * kGroup + wave * 32, left = min(32, kn - key);   // keys past the last read as zero
      const __amdgpu_buffer_rsrc_t r =
          row_rsrc(kbase + (left > 0 ? (int64_t)key * p.kt : 0), left > 0 ? ((int64_t)(left - 1) * p.kt + D) * 2 : 0);
#pragma unroll
      for (int i = 0; i < DMAS; ++i) {
        const int row = (i * 64 + lane) / CH, ch = (i * 64 + lane) % CH ^ (row / RPB % PAIRS) * 2;
        dma16(r, mine + i * 1024, (uint32_t)(row * p.kt * 2 + ch * 16));
      }
    };
    if (g0 < g1) issue(g0);
    // The lane's row; lanes past the last one repeat it and see nothing.
    const int rows = p.q_rows * p.group, r = min(col, rows - 1), tok = p.by_group.of(r), h = hd * p.group + r - tok * p.group;
    const uint16_t* const q = p.q + seq * p.qb + tok * p.qt + h * p.qh;
    V8 qf[KD];
#pragma unroll
    for (int d = 0; d < KD; ++d) qf[d] = *reinterpret_cast<const V8*>(q + 16 * d + 8 * half);
    const float l2 = p.lse[((int64_t)seq * p.q_rows + tok) * p.heads + h] * kLog2e;
    const int lim = col >= rows ? 0 : (p.causal ? hidden + tok + 1 : kn);
    const float* const w = p.w + ((int64_t)seq * p.kv_heads + hd) * p.k_rows;
    float* const out = p.out + ((int64_t)seq * p.kv_heads + hd) * p.k_rows;
    for (int g = g0; g < g1; ++g) {
      const int key0 = g * kGroup + wave * 32;
      // Lane col < 16 of a half has this key in the end.
      const int key = key0 + 8 * (col >> 2) + 4 * half + (col & 3);
      const float had = col < 16 && key < kn ? w[key] : 0.0f;
      __builtin_amdgcn_s_waitcnt(0x70 | 0xf00);   // vmcnt(0): this wave's keys are there
      asm volatile("" ::: "memory");
      V8 kf[KD];
#pragma unroll
      for (int d = 0; d < KD; ++d)
        kf[d] = *reinterpret_cast<const V8*>(mine + col * ROW + ((2 * d + half) ^ (col / RPB % PAIRS) * 2) * 16);
      __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): and in registers
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      if (g + 1 < g1) issue(g + 1);
      v16f s = {};
#pragma unroll
      for (int d = 0; d < KD; ++d) s = Mfma<T>::mul(kf[d], qf[d], s);
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], p.c, -l2));
        const float v = half_sum(key0 + 8 * (e >> 2) + 4 * half + (e & 3) < lim ? x : 0.0f);
        sum = col == e ? v : sum;
      }
      if (col < 16 && key < kn) out[key] = had + sum;
    }
  }
  if (p.out == p.w) return;
  // Places behind the caches' keys stay as they were.
  const int runs = ceil_div(p.k_rows, kCopied);
  for (int64_t i = blockIdx.x; i < (int64_t)p.n * p.kv_heads * runs; i += gridDim.x) {
    const int64_t row = i / runs;
    const int kn = keys_of(p.lengths, (int)(row / p.kv_heads), p.k_rows), from = (int)(i - row * runs) * kCopied;
#pragma unroll
    for (int j = 0; j < kCopied / 256; ++j) {
      const int key = from + 256 * j + (int)threadIdx.x;
      if (key >= kn && key < p.k_rows) p.out[row * p.k_rows + key] = p.w[row * p.k_rows + key];
    }
  }
}

// ------------------------------------------------------------- eviction ----
// Of a cache's n > budget keys stay the last `recent` and, of the others, the
// budget - recent of most weight; of equal weights the first ones. They keep their order.
struct EvictArgs {
  const float* w;          // [n][heads][size]
  const int32_t* lengths;  // or null
  float* w_out;            // [n][heads][capacity]
  int32_t* lengths_out;    // [n]
  int32_t* kept;           // [n][heads][budget]: places in the cache, -1 behind the last
  const char *k, *v;
  char *k_out, *v_out;
  int64_t kt, kh, kb, vt, vh, vb;        // strides of a key, a head, a cache, in bytes
  int64_t kot, koh, kob, vot, voh, vob;
  int n, heads, size, budget, recent, capacity;
  int chunks;              // 16-byte pieces of a row
  int clear;               // whether rows behind a cache's last are set to zero
  uint32_t* hist;          // where parts > 1: counts of three digits [3][n][heads][parts][2048],
  uint4* found;            // and [n][heads][parts] what is known of the border (choose_keys)
  int parts;               // of kPart keys
};

// A weight's place in an order of 32-bit numbers: NaN below all others, -0 like 0.
__device__ __forceinline__ uint32_t order_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);
  return w != w ? 0u : (u & 0x80000000u ? ~u : u | 0x80000000u);
}

constexpr uint32_t kZeroOrder = 0x80000000u;
constexpr int kSelect = 1024;           // threads
constexpr int kEach = 16;               // weights of a thread
constexpr int kPart = kSelect * kEach;  // and of a workgroup
constexpr int kBins = 2048;
constexpr int kDigitShift[3] = {21, 10, 0}, kDigitBits[3] = {11, 11, 10};

// The places that stay, for each cache and head. The border between staying and leaving is found
// digit by digit from the most significant one on, by counting how many weights have each
// value of it; then every weight's place among those that stay is a count of the ones before
// it. A workgroup has 16384 weights, in registers; a wave's are next to each other.
//   WHOLE   a cache of one workgroup: all of it in one kernel
//   0, 1, 2 the border's digit before from its counts, then the counts of this digit, for each
//           workgroup's part
//   PLACE   the last digit, then the places
// (Four caches of 40000 to 131072 keys, 8 heads: a workgroup for each, that went through its weights
// five times, took 159 us; the four kernels take 42.)
constexpr int kPlace = 3, kWhole = 4;

// Sum of the waves' numbers v[0], v[2], .. before wave `end`.
__device__ __forceinline__ uint32_t sum_before(const uint32_t* v, int end) {
  const int lane = threadIdx.x & 63;
  return (uint32_t)__builtin_amdgcn_readlane(wave_prefix_sum(lane < end ? (int)v[2 * lane] : 0), 63);
}

template <int STEP>
__global__ __launch_bounds__(kSelect) void choose_keys(EvictArgs p) {
  constexpr int WAVES = kSelect / 64;
  __shared__ uint32_t bins[kBins];
  __shared__ uint32_t found[2];            // digit, keys above it
  __shared__ uint32_t counts[WAVES][2];    // of a wave: keys above the border, and on it
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int part = blockIdx.x % (uint32_t)p.parts, row = blockIdx.x / (uint32_t)p.parts;
  const int head = row % (uint32_t)p.heads, seq = row / (uint32_t)p.heads;
  const int n = keys_of(p.lengths, seq, p.size);
  const int stay = min(n, p.budget);
  const float* const w = p.w + (int64_t)row * p.size;
  float* const w_out = p.w_out + (int64_t)row * p.capacity;
  int32_t* const kept = p.kept + (int64_t)row * p.budget;
  // The thread's weights: `each`, this one and every 64th on. (Small caches are spread over all waves.)
  const int each = p.parts > 1 ? kEach : (p.size + kSelect - 1) / kSelect;
  const int first = part * kPart + wave * (64 * each) + lane;
  if (STEP >= kPlace && part == 0) {
    if (head == 0 && t == 0) p.lengths_out[seq] = stay;
    for (int i = stay + t; i < p.capacity; i += kSelect) w_out[i] = 0.0f;
    for (int i = stay + t; i < p.budget; i += kSelect) kept[i] = -1;
  }
  if (STEP < kPlace && n <= p.budget) return;
  float x[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) x[j] = j < each && first + 64 * j < n ? w[first + 64 * j] : 0.0f;
  if (n <= p.budget) {
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (j < each && first + 64 * j < n) {
        kept[first + 64 * j] = first + 64 * j;
        w_out[first + 64 * j] = x[j];
      }
    return;
  }
  const int recent = min(p.recent, n), old = n - recent, need = p.budget - recent;   // old > need
  // Weights of this part by digit d, those with the border's digits before it.
  uint32_t border = 0, equals = need;
  auto count = [&](int d) {
    const int shift = kDigitShift[d], bits = kDigitBits[d];
    for (int i = t; i < kBins; i += kSelect) bins[i] = 0;
    __syncthreads();
    int zeros = 0;   // a common weight, which would queue at its bin
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      if (j >= each) break;
      const uint32_t o = order_of(x[j]);
      const bool in = first + 64 * j < old && (d == 0 || o >> (shift + bits) == border >> (shift + bits));
      zeros += in && o == kZeroOrder;
      if (in && o != kZeroOrder) atomicAdd(&bins[o >> shift & ((1u << bits) - 1)], 1u);
    }
    zeros = wave_prefix_sum(zeros);
    if (lane == 63 && zeros) atomicAdd(&bins[kZeroOrder >> shift & ((1u << bits) - 1)], (uint32_t)zeros);
    __syncthreads();
  };
  // The digit at which the counts from the top on reach what is left to stay. Thread t has bins
  // 2047 - 2 t and 2046 - 2 t.
  auto settle = [&](int d, uint32_t c0, uint32_t c1) {
    const uint32_t upto = (uint32_t)wave_prefix_sum((int)(c0 + c1));
    __syncthreads();
    if (lane == 63) counts[wave][0] = upto;
    __syncthreads();
    const uint32_t above = upto - c0 - c1 + sum_before(&counts[0][0], wave);
    if (above < equals && above + c0 >= equals) {
      found[0] = (uint32_t)(kBins - 1 - 2 * t);
      found[1] = above;
    } else if (above + c0 < equals && above + c0 + c1 >= equals) {
      found[0] = (uint32_t)(kBins - 2 - 2 * t);
      found[1] = above + c0;
    }
    __syncthreads();
    border |= found[0] << kDigitShift[d];
    equals -= found[1];
  };
  // The counts of a digit, of part q, at this thread's bins (the upper one in y).
  auto counted = [&](int d, int q) {
    return *reinterpret_cast<const uint2*>(p.hist + (((int64_t)d * p.n * p.heads + row) * p.parts + q) * kBins + kBins - 2 - 2 * t);
  };
  uint32_t before[2] = {0, 0};   // this part: keys above the border, and on it
  if (need == 0) {
    if (STEP < kPlace) return;
    border = 0xffffffffu;   // none
  } else if (STEP == kWhole) {
    for (int d = 0; d < 3; ++d) {
      count(d);
      settle(d, bins[kBins - 1 - 2 * t], bins[kBins - 2 - 2 * t]);
    }
  } else {
    // What the steps before have found: the border's digits, how many on it are left to stay, and
    // the keys of the parts before this one that are above it.
    uint4& known = p.found[(int64_t)row * p.parts + part];
    if constexpr (STEP > 1) {
      border = known.x;
      equals = known.y;
    }
    if constexpr (STEP > 0) {
      constexpr int DIGIT = STEP - 1, COUNT = 8;   // parts on their way at a time
      uint32_t c0 = 0, c1 = 0, mine0 = 0, mine1 = 0;
      for (int q = 0; q < p.parts; q += COUNT) {
        uint2 c[COUNT];
#pragma unroll
        for (int i = 0; i < COUNT; ++i) c[i] = q + i < p.parts ? counted(DIGIT, q + i) : make_uint2(0, 0);
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
          c0 += c[i].y;
          c1 += c[i].x;
          mine0 += q + i < part ? c[i].y : 0;
          mine1 += q + i < part ? c[i].x : 0;
        }
      }
      settle(DIGIT, c0, c1);
      const int digit = (int)found[0], upper = kBins - 1 - 2 * t;   // this thread's bins: upper and the one below
      const uint32_t above = (upper > digit ? mine0 : 0) + (upper - 1 > digit ? mine1 : 0);
      const uint32_t same = (upper == digit ? mine0 : 0) + (upper - 1 == digit ? mine1 : 0);
      // The sums over the threads' bins.
      const uint32_t a = (uint32_t)wave_prefix_sum((int)above), b = (uint32_t)wave_prefix_sum((int)same);
      __syncthreads();
      if (lane == 63) {
        counts[wave][0] = a;
        counts[wave][1] = b;
      }
      __syncthreads();
      before[0] = sum_before(&counts[0][0], WAVES) + (STEP > 1 ? known.z : 0);
      before[1] = sum_before(&counts[0][1], WAVES);
      __syncthreads();   // known has been read
      if (STEP < kPlace && t == 0) known = make_uint4(border, equals, before[0], 0);
    }
    if (STEP < kPlace) {
      count(STEP);
      uint32_t* const to = p.hist + (((int64_t)STEP * p.n * p.heads + row) * p.parts + part) * kBins;
      for (int i = t; i < kBins; i += kSelect) to[i] = bins[i];
      return;
    }
  }
  uint32_t larger = 0, on = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (j >= each) break;
    const uint32_t o = order_of(x[j]);
    const bool in = first + 64 * j < old;
    larger += (uint32_t)__builtin_popcountll(__ballot(in && o > border));
    on += (uint32_t)__builtin_popcountll(__ballot(in && o == border));
  }
  __syncthreads();
  if (lane == 0) {
    counts[wave][0] = larger;
    counts[wave][1] = on;
  }
  __syncthreads();
  larger = before[0] + sum_before(&counts[0][0], wave);
  on = before[1] + sum_before(&counts[0][1], wave);
  const uint64_t below = (1ULL << lane) - 1;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (j >= each) break;
    const int at = first + 64 * j;
    const uint32_t o = order_of(x[j]);
    const bool is_larger = at < old && o > border, is_on = at < old && o == border;
    const uint64_t ml = __ballot(is_larger), mo = __ballot(is_on);
    const uint32_t rank = on + (uint32_t)__builtin_popcountll(mo & below);
    uint32_t to = larger + (uint32_t)__builtin_popcountll(ml & below) + min(rank, equals);
    if (at >= old) to = (uint32_t)(need + at - old);   // the latest come last
    if (is_larger || (is_on && rank < equals) || (at >= old && at < n)) {
      kept[to] = at;
      w_out[to] = x[j];
    }
    larger += (uint32_t)__builtin_popcountll(ml);
    on += (uint32_t)__builtin_popcountll(mo);
  }
}

// Rows of keys and values that stay: a thread moves 16 bytes of each (16384 keys of 8 heads in
// four caches: 92 us, 5.8 TB/s).
__global__ __launch_bounds__(256) void move_rows(EvictArgs p) {
  const uint32_t per_place = (uint32_t)(p.heads * p.chunks), total = (uint32_t)p.budget * per_place;
  const uint32_t blocks = (total + 255) / 256;
  const int seq = (int)(blockIdx.x / blocks);
  const uint32_t i = (blockIdx.x - seq * blocks) * 256 + threadIdx.x;
  if (i >= total) return;
  const int place = (int)(i / per_place), rest = (int)(i - place * per_place);
  const int head = rest / p.chunks, at = (rest - head * p.chunks) * 16;
  const int from = p.kept[((int64_t)seq * p.heads + head) * p.budget + place];
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (from >= 0) {
    k = load_nt(reinterpret_cast<const uint4*>(p.k + seq * p.kb + from * p.kt + head * p.kh + at));
    v = load_nt(reinterpret_cast<const uint4*>(p.v + seq * p.vb + from * p.vt + head * p.vh + at));
  } else if (!p.clear) {
    return;
  }
  store_nt(reinterpret_cast<uint4*>(p.k_out + seq * p.kob + place * p.kot + head * p.koh + at), k);
  store_nt(reinterpret_cast<uint4*>(p.v_out + seq * p.vob + place * p.vot + head * p.voh + at), v);
}

struct WeighPlan {
  int shares;   // of a key head's work (0: a workgroup for every 128 keys)
  int places;   // of pieces for a key head (few rows), else 0
  int64_t grid, join;
  int64_t bytes(int kv_heads) const { return (int64_t)shares * kv_heads * 2 * kDealt * 4; }
};

WeighPlan weigh_plan(int64_t n, int64_t q_rows, int64_t k_rows, int heads, int kv_heads) {
  WeighPlan pl = {};
  const int64_t rows = q_rows * (heads / kv_heads), cus = compute_units(), groups = n * kv_heads * ((k_rows + kGroup - 1) / kGroup);
  if (rows > 0 && rows <= 32 && n <= kListed && n > 0) {
    // Four workgroups per CU are resident; each cache has a piece at least.
    const int64_t places = 4 * cus / kv_heads;
    pl.places = (int)(places < n ? n : places);
    pl.grid = (int64_t)pl.places * kv_heads;
  } else if (rows > 23 * kKeys && groups <= 2 * cus && n <= kShared) {
    // Few workgroups, of 24 tiles of rows and more: dealt out, two resident per CU (40 heads over
    // 8, causal: 1024 tokens 26 us, a workgroup for every 128 keys 79; four times 300 over 2000
    // keys 34 and 36; 256 tokens over 8192 keys, 20 tiles, 39 and 35. 2048 tokens of 40 key
    // heads, 640 workgroups of 32 tiles, 48 and 45; 8 x 2048 tokens, 1024 of 160, 241 and 248).
    pl.shares = 2 * cus / kv_heads > 0 ? (int)(2 * cus / kv_heads) : 1;
    pl.grid = (int64_t)pl.shares * kv_heads;
    pl.join = n * ((k_rows + kDealt - 1) / kDealt) * kv_heads;
  } else {
    pl.grid = groups;
  }
  return pl;
}

template <typename T, int D>
void weigh(const WeighArgs& p, const WeighPlan& pl, hipStream_t s) {
  if (pl.places) weigh_few<T, D><<<(unsigned)pl.grid, 256, 0, s>>>(p);
  else if (pl.shares) weigh_keys<T, D, 2><<<(unsigned)pl.grid, 256, 0, s>>>(p);
  else weigh_keys<T, D, 1><<<(unsigned)pl.grid, 256, 0, s>>>(p);
}

template <typename T>
void weigh_by_dim(const WeighArgs& p, int dim, const WeighPlan& pl, hipStream_t s) {
  if (dim == 32) weigh<T, 32>(p, pl, s);
  else if (dim == 64) weigh<T, 64>(p, pl, s);
  else weigh<T, 128>(p, pl, s);
}

int check_weigh(int64_t n, int64_t q_rows, int64_t k_rows, int heads, int kv_heads, int head_dim) {
  LR_REQUIRE(n >= 0 && q_rows >= 0 && k_rows >= 0, "attention_weights: negative shape");
  LR_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0,
             "attention_weights: %d heads do not share %d key heads evenly", heads, kv_heads);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(LR_EUNSUPPORTED, "attention_weights: head_dim %d is not supported (32, 64 or 128)", head_dim);
  LR_REQUIRE(n < (1LL << 24) && q_rows < (1LL << 30) && k_rows < (1LL << 30) && heads <= 65536,
             "attention_weights: shapes past 2^24 sequences, 2^30 rows or 65536 heads are not supported");
  LR_REQUIRE(q_rows * (heads / kv_heads) < (1LL << 30), "attention_weights: %lld rows of a key head are not supported",
             (long long)(q_rows * (heads / kv_heads)));
  LR_REQUIRE(k_rows == 0 || n < (1LL << 40) / k_rows / kv_heads, "attention_weights: %lld caches of %lld keys are not supported",
             (long long)n, (long long)k_rows);
  return LR_OK;
}

}  // namespace
}  // namespace lr

using namespace lr;

extern "C" int lr_attention_weights_workspace(int64_t sequences, int64_t q_rows, int64_t k_rows, int heads, int kv_heads,
                                              int head_dim, int64_t* bytes) {
  if (int rc = check_weigh(sequences, q_rows, k_rows, heads, kv_heads, head_dim)) return rc;
  LR_REQUIRE(bytes, "attention_weights: null pointer");
  *bytes = weigh_plan(sequences, q_rows, k_rows, heads, kv_heads).bytes(kv_heads);
  return LR_OK;
}

extern "C" int lr_attention_weights(const void* q, const void* k, const float* lse, const float* weights, float* out,
                                    int dtype, int64_t sequences, int64_t q_rows, int64_t k_rows, int heads,
                                    int kv_heads, int head_dim, const int64_t* strides, const int32_t* key_lengths,
                                    int causal, int scale_bits, void* workspace, int64_t workspace_bytes, void* stream) {
  LR_REQUIRE(dtype == LR_DTYPE_BF16 || dtype == LR_DTYPE_F16, "attention_weights: unknown dtype %d", dtype);
  if (int rc = check_weigh(sequences, q_rows, k_rows, heads, kv_heads, head_dim)) return rc;
  if (sequences == 0 || k_rows == 0) return LR_OK;
  LR_REQUIRE(k && weights && out && strides && (q_rows == 0 || (q && lse)), "attention_weights: null pointer");
  LR_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(lse, 4) && aligned(weights, 4) && aligned(out, 4),
             "attention_weights: queries and keys must be 16-byte aligned, sums and weights 4-byte");
  for (int i = 0; i < 6; ++i)
    LR_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0,
               "attention_weights: stride %d is %lld, not a multiple of 8 from 0 on", i, (long long)strides[i]);
  const int group = heads / kv_heads;
  // A tile's keys and queries are addressed by 32-bit byte offsets from its first one.
  LR_REQUIRE(strides[3] < (1LL << 23), "attention_weights: strides of 2^23 and more between keys are not supported");
  LR_REQUIRE((group == 1 || strides[1] < (1LL << 30) / group) && strides[0] < (1LL << 29) / kKeys,
             "attention_weights: queries of a key head and tile more than 2^31 bytes apart are not supported");
  float scale;
  static_assert(sizeof scale == sizeof scale_bits, "fp32");
  __builtin_memcpy(&scale, &scale_bits, sizeof scale);
  const WeighPlan pl = weigh_plan(sequences, q_rows, k_rows, heads, kv_heads);
  const WeighArgs p = {static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), lse, weights, out,
                       static_cast<float*>(workspace), strides[0], strides[1], strides[2], strides[3], strides[4],
                       strides[5], key_lengths, (int)sequences, (int)q_rows, (int)k_rows, heads, kv_heads, group,
                       causal != 0, pl.shares, pl.places, scale * 1.4426950408889634f, 1.0f / (float)group, Divisor((uint32_t)group)};
  LR_REQUIRE(p.c > 0.0f && isfinite(p.c), "attention_weights: the scale must be positive and finite");
  LR_REQUIRE(pl.grid <= kMaxBlocks && pl.join <= kMaxBlocks, "attention_weights: %lld workgroups are not supported",
             (long long)(pl.grid > pl.join ? pl.grid : pl.join));
  LR_REQUIRE(pl.shares == 0 || (workspace && aligned(workspace, 4) && workspace_bytes >= pl.bytes(kv_heads)),
             "attention_weights: needs a workspace of %lld bytes", (long long)pl.bytes(kv_heads));
  hipStream_t s = as_stream(stream);
  if (dtype == LR_DTYPE_BF16) weigh_by_dim<__bf16>(p, head_dim, pl, s);
  else weigh_by_dim<_Float16>(p, head_dim, pl, s);
  if (int rc = check_launch("attention_weights")) return rc;
  if (pl.shares == 0) return LR_OK;
  join_shares<<<(unsigned)pl.join, kDealt, 0, s>>>(p);
  return check_launch("attention_weights");
}

static int64_t evict_bytes(int64_t sequences, int64_t size, int kv_heads) {
  return size > kPart ? sequences * kv_heads * ((size + kPart - 1) / kPart) * (3 * kBins * 4 + 16) : 0;
}

extern "C" int lr_cache_evict_workspace(int64_t sequences, int64_t size, int kv_heads, int64_t* bytes) {
  LR_REQUIRE(sequences >= 0 && sequences < (1LL << 24) && size >= 0 && size < (1LL << 30) && kv_heads > 0 &&
                 kv_heads <= 65536,
             "cache_evict: %lld caches of %lld keys are not supported", (long long)sequences, (long long)size);
  LR_REQUIRE(bytes, "cache_evict: null pointer");
  *bytes = evict_bytes(sequences, size, kv_heads);
  return LR_OK;
}

extern "C" int lr_cache_evict(const void* k, const void* v, const float* weights, const int32_t* key_lengths, void* k_out,
                              void* v_out, float* weights_out, int32_t* lengths_out, int32_t* kept, int64_t sequences,
                              int64_t size, int kv_heads, int64_t row_bytes, int64_t budget, int64_t recent,
                              int64_t capacity, const int64_t* strides, int clear, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  LR_REQUIRE(sequences >= 0 && size >= 0 && kv_heads > 0 && row_bytes > 0, "cache_evict: negative shape");
  LR_REQUIRE(budget > 0 && recent >= 0 && recent <= budget && capacity >= budget,
             "cache_evict: a budget of %lld, %lld of them the latest, in caches of %lld", (long long)budget,
             (long long)recent, (long long)capacity);
  if (sequences == 0) return LR_OK;
  LR_REQUIRE(row_bytes % 16 == 0 && row_bytes <= (1 << 20), "cache_evict: rows of %lld bytes, not a multiple of 16",
             (long long)row_bytes);
  LR_REQUIRE(sequences < (1LL << 24) && size < (1LL << 30) && capacity < (1LL << 30) && kv_heads <= 65536,
             "cache_evict: shapes past 2^24 caches, 2^30 keys or 65536 heads are not supported");
  LR_REQUIRE((k && v && weights) || size == 0, "cache_evict: null pointer");
  LR_REQUIRE(k_out && v_out && weights_out && lengths_out && kept && strides, "cache_evict: null pointer");
  LR_REQUIRE(aligned(k, 16) && aligned(v, 16) && aligned(k_out, 16) && aligned(v_out, 16) && aligned(weights, 4) &&
                 aligned(weights_out, 4) && aligned(lengths_out, 4) && aligned(kept, 4),
             "cache_evict: keys and values must be 16-byte aligned");
  for (int i = 0; i < 12; ++i)
    LR_REQUIRE(strides[i] >= 0 && strides[i] % 16 == 0,
               "cache_evict: stride %d is %lld bytes, not a multiple of 16 from 0 on", i, (long long)strides[i]);
  const int64_t chunks = row_bytes / 16, moved = budget * kv_heads * chunks;
  const int64_t blocks = (moved + 255) / 256 * sequences;
  const int64_t parts = size > kPart ? (size + kPart - 1) / kPart : 1;
  LR_REQUIRE(moved < (1LL << 31) && blocks <= kMaxBlocks && sequences * kv_heads * parts <= kMaxBlocks / 4,
             "cache_evict: %lld rows of %lld caches are not supported", (long long)(budget * kv_heads),
             (long long)sequences);
  const int64_t needs = evict_bytes(sequences, size, kv_heads);
  LR_REQUIRE(needs == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= needs),
             "cache_evict: needs a workspace of %lld bytes", (long long)needs);
  const EvictArgs p = {weights, key_lengths, weights_out, lengths_out, kept, static_cast<const char*>(k),
                       static_cast<const char*>(v), static_cast<char*>(k_out), static_cast<char*>(v_out), strides[0],
                       strides[1], strides[2], strides[3], strides[4], strides[5], strides[6], strides[7], strides[8],
                       strides[9], strides[10], strides[11], (int)sequences, kv_heads, (int)size, (int)budget,
                       (int)recent, (int)capacity, (int)chunks, clear != 0, static_cast<uint32_t*>(workspace),
                       reinterpret_cast<uint4*>(static_cast<uint32_t*>(workspace) + 3 * sequences * kv_heads * parts * kBins),
                       (int)parts};
  hipStream_t s = as_stream(stream);
  const unsigned grid = (unsigned)(sequences * kv_heads * parts);
  if (parts == 1) {
    choose_keys<kWhole><<<grid, kSelect, 0, s>>>(p);
  } else {
    choose_keys<0><<<grid, kSelect, 0, s>>>(p);
    if (int rc = check_launch("cache_evict")) return rc;
    choose_keys<1><<<grid, kSelect, 0, s>>>(p);
    if (int rc = check_launch("cache_evict")) return rc;
    choose_keys<2><<<grid, kSelect, 0, s>>>(p);
    if (int rc = check_launch("cache_evict")) return rc;
    choose_keys<kPlace><<<grid, kSelect, 0, s>>>(p);
  }
  if (int rc = check_launch("cache_evict")) return rc;
  move_rows<<<(unsigned)blocks, 256, 0, s>>>(p);
  return check_launch("cache_evict");
}
