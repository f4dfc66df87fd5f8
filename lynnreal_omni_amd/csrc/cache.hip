// cache.hip - caches of bounded size: the attention weight that each key gets, and the
// choice of the keys that stay.
//
// Weights. With the logarithm of each row's softmax sum given, a key j of key head h gets
//   w[j] += sum over rows r of h that see j of exp(scale q_r . k_j - lse_r),
// rows being tokens x the query heads that share h. A sum over rows per key is the
// transpose of what attention does, so a workgroup keeps keys, in registers, and the
// queries go by: S^T = K Q^T on the 32x32x16 MFMA leaves a lane with 16 keys of one query,
// each added to its own fp32 sum; the sums over the 32 lanes come once at the end. Every
// key is read once, and the order of additions does not depend on timing.
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
  float* part;            // sums of splits of the rows [splits][n][kv_heads][k_rows]
  int64_t qt, qh, qb, kt, kh, kb;
  const int32_t* lengths;
  int n, q_rows, k_rows, heads, kv_heads, group;
  int causal, splits;     // splits: of the rows, `chunk` tiles of 64 each
  int chunk;
  int places;             // few rows: pieces of all caches for a key head
  float c;                // scale * log2(e)
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

// Four waves with KB blocks of 32 keys each; queries in tiles of 64 rows, with their sums,
// through a ring in the LDS that first holds the keys on their way to the registers. Swizzle as
// in lr_attention.h.
template <typename T, int D, int KB>
__global__ __launch_bounds__(256, 2) void weigh_keys(WeighArgs p) {
  typedef typename Mfma<T>::V V8;
  constexpr int ROW = 2 * D, CH = ROW / 16, RPB = 256 / ROW, PAIRS = ROW / 32, KD = D / 16;
  constexpr int WAVES = 4, TILE = kKeys * ROW, DMAS = TILE / 1024 / WAVES, KEYS = 32 * WAVES * KB;
  constexpr int RING = KEYS / kKeys, LOADS = DMAS + 1;   // slots that fit into the keys' LDS; DMAs per wave and tile
  // (One array for all of it: between two the compiler waits for every DMA before any read.)
  __shared__ __attribute__((aligned(1024))) char smem[KEYS * (ROW + 4) + RING * WAVES * kKeys * 4];
  float* const sums = reinterpret_cast<float*>(smem + KEYS * ROW);
  char* const lses = smem + KEYS * (ROW + 4);   // [RING][WAVES][64], each wave's own
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int half = lane >> 5, col = lane & 31;
  // Heads, which lie side by side, first; then sequences, so that the first keys, which
  // the most rows see where causal, come first.
  uint32_t id = blockIdx.x;
  const int hd = (int)(id % (uint32_t)p.kv_heads);
  id /= (uint32_t)p.kv_heads;
  const int seq = (int)(id % (uint32_t)p.n);
  id /= (uint32_t)p.n;
  const int split = (int)(id % (uint32_t)p.splits), key0 = (int)(id / (uint32_t)p.splits) * KEYS;
  const int kn = keys_of(p.lengths, seq, p.k_rows);
  const int hidden = kn - p.q_rows;   // causal: token t sees keys up to hidden + t
  const int rows = p.q_rows * p.group;
  const int first = p.causal ? (int)min((int64_t)rows, max(0, key0 - hidden) * (int64_t)p.group) : 0;
  const int tiles = key0 < kn ? (rows - first + kKeys - 1) / kKeys : 0;
  // Splits of one size, whatever the keys' own number of rows: causal ones are then as long.
  const int t0 = min(tiles, split * p.chunk), t1 = min(tiles, t0 + p.chunk);
  float acc[KB][16];
#pragma unroll
  for (int b = 0; b < KB; ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[b][e] = 0.0f;
  if (t0 < t1) {
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
    for (int g = 0; g < KEYS / kKeys; ++g) {
      const int left = min(kKeys, kn - key0 - g * kKeys);   // keys past the last read as zero
      const __amdgpu_buffer_rsrc_t r = row_rsrc(kbase + (key0 + (int64_t)g * kKeys) * p.kt,
                                                left > 0 ? ((int64_t)(left - 1) * p.kt + D) * 2 : 0);
#pragma unroll
      for (int i = 0; i < DMAS; ++i)
        dma16(r, smem + g * TILE + (wave * DMAS + i) * 1024, (uint32_t)(slot_row(i) * p.kt * 2 + slot_chunk(i) * 16));
    }
    publish(std::integral_constant<int, 0>{});
    V8 kf[KB][KD];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const int row = (wave * KB + b) * 32 + col;
#pragma unroll
      for (int d = 0; d < KD; ++d)
        kf[b][d] = *reinterpret_cast<const V8*>(smem + row * ROW + ((2 * d + half) ^ (row / RPB % PAIRS) * 2) * 16);
    }
    __syncthreads();   // the keys are in registers: the queries may take their place
    const uint16_t* const qbase = p.q + seq * p.qb + (int64_t)hd * p.group * p.qh;
    const float* const lbase = p.lse + (int64_t)seq * p.q_rows * p.heads + hd * p.group;
    // Rows past the last one repeat it and are masked; tiles past the last one, which keep
    // the count of loads the same, repeat that.
    auto issue = [&](int t) {
      const int slot = (t - t0) % RING, r0 = first + min(t, t1 - 1) * kKeys, tok0 = p.by_group.of(r0);
      const int toks = min(kKeys, p.q_rows - tok0);   // that 64 rows from r0 on can have
      const __amdgpu_buffer_rsrc_t rs =
          row_rsrc(qbase + (int64_t)tok0 * p.qt, ((toks - 1) * p.qt + (p.group - 1) * p.qh + D) * 2);
#pragma unroll
      for (int i = 0; i < DMAS; ++i) {
        const int r = min(r0 + slot_row(i), rows - 1), tok = p.by_group.of(r);
        dma16(rs, smem + slot * TILE + (wave * DMAS + i) * 1024,
              (uint32_t)((tok - tok0) * p.qt * 2 + (r - tok * p.group) * p.qh * 2 + slot_chunk(i) * 16));
      }
      const __amdgpu_buffer_rsrc_t ls =
          row_rsrc(lbase + (int64_t)tok0 * p.heads, ((int64_t)(toks - 1) * p.heads + p.group) * 4);
      const int r = min(r0 + lane, rows - 1), tok = p.by_group.of(r);
      dma4(ls, lses + (slot * WAVES + wave) * kKeys * 4, (uint32_t)(((tok - tok0) * p.heads + r - tok * p.group) * 4));
    };
    // Adds a block's shares, which are those of keys past `lim` too where WHOLE. lim counts from
    // the lane's first key on.
    const int own = key0 + wave * KB * 32 + 4 * half;
    auto add = [&](const v16f (&s)[KB], float l2, int lim, int x, int e, auto whole) __attribute__((always_inline)) {
      const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][e], p.c, -l2));
      acc[x][e] += decltype(whole)::value || 32 * x + 8 * (e >> 2) + (e & 3) < lim ? w : 0.0f;
    };
    // The scores of block b of a tile, while the exponentials of the block before, which every
    // row sees whole, run between the matrix instructions.
    auto product = [&](v16f (&s)[KB], const char* qs, int b, const v16f (&before)[KB], float l2) __attribute__((always_inline)) {
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
        for (int x = 0; x < KB; ++x) s[x] = Mfma<T>::mul(kf[x][d], qf[d & 3], d ? s[x] : zero);
#pragma unroll
        for (int i = 16 * KB * d / KD; i < 16 * KB * (d + 1) / KD; ++i) add(before, l2, 0, i / 16, i % 16, std::true_type{});
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // A block without shares, for the start and behind one that was not whole.
    v16f s0[KB] = {}, s1[KB] = {};
    float l2 = INFINITY;   // of the block before
    auto block = [&](v16f (&s)[KB], v16f (&before)[KB], const char* qs, int t, int b, float sum2, int lim) __attribute__((always_inline)) {
      product(s, qs, b, before, l2);
      l2 = sum2;
      const int r0 = first + t * kKeys + 32 * b;
      if (r0 + 32 <= rows && (!p.causal || hidden + p.by_group.of(r0) + 1 >= key0 + KEYS)) return;
#pragma unroll
      for (int x = 0; x < KB; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          add(s, l2, lim, x, e, std::false_type{});
          s[x][e] = 0.0f;
        }
      l2 = INFINITY;
    };
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) issue(t0 + i);
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      publish(std::integral_constant<int, (RING - 2) * LOADS>{});   // tile t; every wave is done with tile t - 1
      issue(t + RING - 1);
      const int slot = (t - t0) % RING;
      const char* const qs = smem + slot * TILE;
      // Of the lane's row in each block: lse * log2(e), and the keys that it sees.
      float now[2];
      int lim[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        now[b] = reinterpret_cast<const float*>(lses)[(slot * WAVES + wave) * kKeys + 32 * b + col] * kLog2e;
        const int r = first + t * kKeys + 32 * b + col;
        lim[b] = r >= rows ? 0 : (p.causal ? hidden + p.by_group.of(r) + 1 : kn) - own;
      }
      block(s0, s1, qs, t, 0, now[0], lim[0]);
      if (first + t * kKeys + 32 >= rows) {   // the last tile, without a second block
#pragma unroll
        for (int x = 0; x < KB; ++x)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            add(s0, l2, 0, x, e, std::true_type{});
            s1[x][e] = 0.0f;
          }
        l2 = INFINITY;
        break;
      }
      block(s1, s0, qs, t, 1, now[1], lim[1]);
    }
#pragma unroll
    for (int x = 0; x < KB; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) add(s1, l2, 0, x, e, std::true_type{});
  }
  __builtin_amdgcn_s_waitcnt(0x70 | 0xf00);   // the last DMAs have landed before the LDS goes to another
#pragma unroll
  for (int x = 0; x < KB; ++x)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float v = half_sum(acc[x][e]);
      if (col == 0) sums[(wave * KB + x) * 32 + 8 * (e >> 2) + 4 * half + (e & 3)] = v;
    }
  __syncthreads();
  const int64_t at = ((int64_t)seq * p.kv_heads + hd) * p.k_rows + key0;
  for (int i = threadIdx.x; i < KEYS; i += 256) {
    if (key0 + i >= p.k_rows) return;
    // Places behind the cache's keys stay as they were.
    if (p.splits > 1) p.part[(int64_t)split * p.n * p.kv_heads * p.k_rows + at + i] = key0 + i < kn ? sums[i] : 0.0f;
    else p.out[at + i] = key0 + i < kn ? p.w[at + i] + sums[i] : p.w[at + i];
  }
}

// At most 32 rows per key head: what counts is the stream of keys. They are cut into pieces
// over all caches (lr_pieces.h); a wave has 32 keys of each 128 of them, through 32 rows of
// LDS of its own, and the queries in registers, so that no wave waits for another. The next
// keys are on their way while these are worked on.
// (Eight caches of 16152 keys in all, places for 65536, 40 heads over 8: 17.2 us with a workgroup
// for every 128 places of every cache.)
constexpr int kGroup = 128;
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

// out = w + the splits' sums, in order.
__global__ __launch_bounds__(256) void add_splits(const float* part, const float* w, float* out, int64_t n, int splits) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float v = part[i];
  for (int s = 1; s < splits; ++s) v += part[s * n + i];
  out[i] = w[i] + v;
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
  uint32_t* hist;          // counts of three digits [3][n][heads][parts][2048], where parts > 1
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
//   0, 1, 2 counts of that digit, for each workgroup's part, into p.hist
//   PLACE   the border and the parts before this one from those counts, then the places
// (Four caches of 40000 to 131072 keys, 8 heads: a workgroup for each, that went through its weights
// five times, took 159 us.)
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
    // All digits' counts first: their loads wait for none of them.
    constexpr int DIGITS = STEP < kPlace ? STEP : 3, COUNT = 8;   // parts on their way at a time
    uint32_t c0[DIGITS + 1] = {}, c1[DIGITS + 1] = {}, mine0[DIGITS + 1] = {}, mine1[DIGITS + 1] = {};
    for (int q = 0; q < p.parts; q += COUNT) {
      uint2 c[DIGITS + 1][COUNT];
#pragma unroll
      for (int d = 0; d < DIGITS; ++d)
#pragma unroll
        for (int i = 0; i < COUNT; ++i) c[d][i] = q + i < p.parts ? counted(d, q + i) : make_uint2(0, 0);
#pragma unroll
      for (int d = 0; d < DIGITS; ++d)
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
          c0[d] += c[d][i].y;
          c1[d] += c[d][i].x;
          mine0[d] += q + i < part ? c[d][i].y : 0;
          mine1[d] += q + i < part ? c[d][i].x : 0;
        }
    }
#pragma unroll
    for (int d = 0; d < DIGITS; ++d) {
      settle(d, c0[d], c1[d]);
      const int digit = (int)found[0], mine = kBins - 1 - 2 * t;
      before[0] += (mine > digit ? mine0[d] : 0) + (mine - 1 > digit ? mine1[d] : 0);
      if (d == 2) before[1] = (mine == digit ? mine0[d] : 0) + (mine - 1 == digit ? mine1[d] : 0);
    }
    if (STEP < kPlace) {
      count(STEP);
      uint32_t* const to = p.hist + (((int64_t)STEP * p.n * p.heads + row) * p.parts + part) * kBins;
      for (int i = t; i < kBins; i += kSelect) to[i] = bins[i];
      return;
    }
    // The sums over the threads' bins.
    const uint32_t a = (uint32_t)wave_prefix_sum((int)before[0]), b = (uint32_t)wave_prefix_sum((int)before[1]);
    __syncthreads();
    if (lane == 63) {
      counts[wave][0] = a;
      counts[wave][1] = b;
    }
    __syncthreads();
    before[0] = sum_before(&counts[0][0], WAVES);
    before[1] = sum_before(&counts[0][1], WAVES);
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

// Rows of keys and values that stay: a thread moves 16 bytes of each.
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
  int blocks, splits, chunk;   // of 32 keys per wave; of the rows, and their tiles
  int places;                  // of pieces for a key head (few rows), else 0
  int64_t grid;
};

WeighPlan weigh_plan(int64_t n, int64_t q_rows, int64_t k_rows, int heads, int kv_heads, bool causal) {
  WeighPlan pl;
  const int64_t rows = q_rows * (heads / kv_heads), tiles = (rows + kKeys - 1) / kKeys, cus = compute_units();
  auto groups_of = [&](int blocks) { return n * kv_heads * ((k_rows + 128 * blocks - 1) / (128 * blocks)); };
  // 64 keys per wave halve what the queries' fragments take of the LDS. With a tile or two of
  // queries the keys' stream counts, and smaller workgroups; so with too few to fill the GPU.
  pl.blocks = tiles > 2 && groups_of(2) * ((tiles + 3) / 4) >= cus ? 2 : 1;
  const int64_t groups = groups_of(pl.blocks);
  // Rows are split, in runs of four tiles and more, for four workgroups per CU, of which two
  // are resident; where causal, half of the runs have no rows and the others differ, for twelve
  // (3683 tokens, 40 heads over 8: 153 us with twelve, 183 with four; all keys 179 with
  // four, 200 with twelve).
  int64_t s = groups > 0 ? (causal ? 12 : 4) * cus / groups : 1;
  if (s > tiles / 4) s = tiles / 4;
  if (s < 1) s = 1;
  if (s > 64) s = 64;
  pl.chunk = (int)((tiles + s - 1) / s);
  pl.splits = pl.chunk > 0 ? (int)((tiles + pl.chunk - 1) / pl.chunk) : 1;
  pl.grid = groups * pl.splits;
  pl.places = 0;
  if (rows > 0 && rows <= 32 && n <= kListed && n > 0) {
    // Four workgroups per CU are resident; each cache has a piece at least.
    const int64_t places = 4 * cus / kv_heads;
    pl.places = (int)(places < n ? n : places);
    pl.splits = 1;
    pl.grid = (int64_t)pl.places * kv_heads;
  }
  return pl;
}

template <typename T, int D>
void weigh(const WeighArgs& p, const WeighPlan& pl, hipStream_t s) {
  if (pl.places) weigh_few<T, D><<<(unsigned)pl.grid, 256, 0, s>>>(p);
  else if (pl.blocks == 1) weigh_keys<T, D, 1><<<(unsigned)pl.grid, 256, 0, s>>>(p);
  else weigh_keys<T, D, 2><<<(unsigned)pl.grid, 256, 0, s>>>(p);
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
                                              int head_dim, int causal, int64_t* bytes) {
  if (int rc = check_weigh(sequences, q_rows, k_rows, heads, kv_heads, head_dim)) return rc;
  LR_REQUIRE(bytes, "attention_weights: null pointer");
  const WeighPlan pl = weigh_plan(sequences, q_rows, k_rows, heads, kv_heads, causal != 0);
  *bytes = pl.splits > 1 ? pl.splits * sequences * kv_heads * k_rows * 4 : 0;
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
  const WeighPlan pl = weigh_plan(sequences, q_rows, k_rows, heads, kv_heads, causal != 0);
  const WeighArgs p = {static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), lse, weights, out,
                       static_cast<float*>(workspace), strides[0], strides[1], strides[2], strides[3], strides[4],
                       strides[5], key_lengths, (int)sequences, (int)q_rows, (int)k_rows, heads, kv_heads, group,
                       causal != 0, pl.splits, pl.chunk, pl.places, scale * 1.4426950408889634f, Divisor((uint32_t)group)};
  LR_REQUIRE(p.c > 0.0f && isfinite(p.c), "attention_weights: the scale must be positive and finite");
  const int64_t all = sequences * kv_heads * k_rows;
  LR_REQUIRE(pl.grid <= kMaxBlocks && (pl.splits == 1 || all <= kMaxBlocks * 256),
             "attention_weights: %lld workgroups are not supported", (long long)pl.grid);
  if (pl.splits > 1)
    LR_REQUIRE(workspace && aligned(workspace, 4) && workspace_bytes >= pl.splits * all * 4,
               "attention_weights: needs a workspace of %lld bytes", (long long)(pl.splits * all * 4));
  hipStream_t s = as_stream(stream);
  if (dtype == LR_DTYPE_BF16) weigh_by_dim<__bf16>(p, head_dim, pl, s);
  else weigh_by_dim<_Float16>(p, head_dim, pl, s);
  if (int rc = check_launch("attention_weights")) return rc;
  if (pl.splits == 1) return LR_OK;
  add_splits<<<(unsigned)((all + 255) / 256), 256, 0, s>>>(p.part, weights, out, all, pl.splits);
  return check_launch("attention_weights");
}

static int64_t evict_bytes(int64_t sequences, int64_t size, int kv_heads) {
  return size > kPart ? 3 * sequences * kv_heads * ((size + kPart - 1) / kPart) * kBins * 4 : 0;
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
