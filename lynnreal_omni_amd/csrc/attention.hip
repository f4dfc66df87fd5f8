// attention.hip - softmax(scale * Q K^T) V for bf16 and fp16, head_dim 32, 64, 128.
//
// One pass over the keys with a running maximum m and sum l per query row:
//   s = scale * q . k;  m' = max(m, s);  p = 2^(log2(e) (s - m'));
//   l = l 2^(log2(e) (m - m')) + sum p;  o = o 2^(log2(e) (m - m')) + p V
// and o / l at the end (0 where a row sees no key). Scores, m, l and o are fp32;
// p is rounded to the inputs' type for the second product (l adds the unrounded
// p), and o / l once at the end.
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
#include <math.h>

#include "lr_device.h"
#include "lr_runtime.h"

namespace lr {
namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));

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
  int heads, kv_heads, group;   // group = heads / kv_heads
  int pack;              // query heads that share a tile's rows (group or 1)
  int causal, splits;
  float c;               // scale * log2(e)
  int64_t tiles;         // row tiles per head in all
};

// A sequence's rows and keys. Values read from the device are clamped, so that
// wrong ones cannot lead outside the tensors.
struct Seq {
  int64_t q0, k0;  // first row / key (token index into q and k, before the batch stride)
  int64_t b;       // dense: sequence
  int qn, kn;
};

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

// Packed rows: sequence i = 0 stands for the rows before cu_q[0], n + 1 for those
// behind cu_q[n]; both have no keys.
__device__ __forceinline__ int64_t first_row(const AttnArgs& p, int64_t i) {
  return i == 0 ? 0 : (i == p.n + 2 ? p.q_rows : clamp64(p.cu_q[i - 1], 0, p.q_rows));
}

template <typename T> struct Mfma;
template <> struct Mfma<__bf16> {
  typedef v8bf V;
  static __device__ __forceinline__ v16f mul(const V& a, const V& b, const v16f& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf2(a, b); }
};
template <> struct Mfma<_Float16> {
  typedef v8h V;
  static __device__ __forceinline__ v16f mul(const V& a, const V& b, const v16f& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const v2h h = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, h);
  }
};

__device__ __forceinline__ float max_with_partner(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_partner(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef __attribute__((address_space(3))) v4s* lds_v4s_t;

// Device-only: the host pass of a kernel's lambdas must not see the builtin.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rsrc, void* lds, uint32_t voffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)lds, 16, voffset, 0, 0, 0);
}

constexpr int kKeys = 64;        // keys per tile
constexpr float kSlack = 8.0f;   // log2

// Rows of a workgroup: 32 * QB per wave. Keys in tiles of 64 through a ring of S
// slots in LDS (K rows, then V rows), by 16-byte DMA. A row's 16-byte chunk c lies
// in slot c ^ 2 * (row / (256 / row bytes) % (row bytes / 32)): eight rows' equal
// 32-byte columns are on distinct banks, which is what both reads need.
template <typename T, int D, int QB, int WAVES, int S>
__global__ __launch_bounds__(64 * WAVES, 1) void attention(AttnArgs p) {
  typedef typename Mfma<T>::V V8;
  constexpr int BM = 32 * QB * WAVES;
  constexpr int ROW = 2 * D;                     // bytes of a row
  constexpr int CH = ROW / 16;                   // chunks per row
  constexpr int RPB = 256 / ROW, PAIRS = ROW / 32;
  constexpr int TILE = kKeys * ROW, SLOT = 2 * TILE;
  constexpr int DMAS = TILE / 1024 / WAVES;      // per wave, operand and tile
  constexpr int KD = D / 16, DB = D / 32;
  static_assert(TILE / 1024 % WAVES == 0, "DMA split");
  __shared__ __attribute__((aligned(1024))) char smem[S * SLOT];
  // fp16 p is kept 2^7 larger: its subnormals then begin at 2^-31 of a row's largest.
  constexpr float kShift = __is_same(T, _Float16) ? 7.0f : 0.0f;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int half = lane >> 5, col = lane & 31;
  // Tiles of a head lie together, and each XCD (workgroups are dealt to them in
  // turn) takes a contiguous run, so that its L2 serves a head's keys once.
  const int64_t total = p.tiles * (p.heads / p.pack) * p.splits;
  const int64_t pid = blockIdx.x;
  const int64_t per = total >> 3, rest = total & 7, xcd = pid & 7;
  const int64_t lid = (xcd < rest ? xcd * (per + 1) : rest * (per + 1) + (xcd - rest) * per) + (pid >> 3);
  const int split = (int)(lid % p.splits);
  int64_t tile = lid / p.splits % p.tiles;
  const int hd = (int)(lid / p.splits / p.tiles);   // head, or key head where heads share rows
  const int kv_head = p.pack > 1 ? hd : hd / p.group;

  Seq s = {};
  if (p.cu_q) {
    // Sequence i has the tile slots from first_row(i) * pack / BM + i on: at least
    // as many as its rows need, and its own.
    const int64_t slot = tile;
    int64_t lo = 0, hi = p.n + 1;
    while (lo < hi) {
      const int64_t mid = (lo + hi + 1) >> 1;
      if (first_row(p, mid) * p.pack / BM + mid <= slot) lo = mid;
      else hi = mid - 1;
    }
    s.q0 = first_row(p, lo);
    s.qn = (int)clamp64(first_row(p, lo + 1) - s.q0, 0, p.q_rows);
    tile = slot - (s.q0 * p.pack / BM + lo);
    if (lo > 0 && lo <= p.n) {
      s.k0 = clamp64(p.cu_k[lo - 1], 0, p.k_rows);
      s.kn = (int)clamp64(clamp64(p.cu_k[lo], 0, p.k_rows) - s.k0, 0, p.k_rows);
    }
  } else {
    const int64_t per_seq = p.tiles / p.n;
    s.b = tile / per_seq;
    tile -= s.b * per_seq;
    s.qn = (int)p.q_rows;
    s.kn = (int)(p.lengths ? clamp64(p.lengths[s.b], 0, p.k_rows) : p.k_rows);
    // Causal: the last tiles see the most keys and go first.
    if (p.causal) tile = per_seq - 1 - tile;
  }
  const int64_t rows = (int64_t)s.qn * p.pack;
  const int64_t r0 = tile * BM;
  if (r0 >= rows) return;

  // This wave's query rows: row r is token r / pack, head hd * pack + r % pack.
  int tok[QB], head[QB];
  int64_t qoff[QB];
  int limit[QB];  // keys that the row sees
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const int64_t r = r0 + wave * 32 * QB + 32 * b + col;
    const int64_t rc = r < rows ? r : rows - 1;
    tok[b] = (int)(p.pack == 1 ? rc : rc / p.pack);
    head[b] = p.pack == 1 ? hd : hd * p.pack + (int)(rc - (int64_t)tok[b] * p.pack);
    qoff[b] = s.b * p.qb + (s.q0 + tok[b]) * p.qt + head[b] * p.qh;
    limit[b] = p.causal ? min(s.kn, max(0, s.kn - s.qn + tok[b] + 1)) : s.kn;
  }
  V8 q[QB][KD];
#pragma unroll
  for (int b = 0; b < QB; ++b)
#pragma unroll
    for (int d = 0; d < KD; ++d)
      q[b][d] = *reinterpret_cast<const V8*>(p.q + qoff[b] + 16 * d + 8 * half);

  // Key tiles [t0, t1) of this split; the last one that any row of the workgroup sees.
  const int64_t last = r0 + BM <= rows ? r0 + BM - 1 : rows - 1;
  const int last_tok = (int)(p.pack == 1 ? last : last / p.pack);
  const int first_tok = (int)(p.pack == 1 ? r0 : r0 / p.pack);
  const int seen = p.causal ? min(s.kn, max(0, s.kn - s.qn + last_tok + 1)) : s.kn;
  const int sure = p.causal ? min(s.kn, max(0, s.kn - s.qn + first_tok + 1)) : s.kn;  // seen by every row
  const int tiles_k = (seen + kKeys - 1) / kKeys;
  const int t0 = (int)((int64_t)tiles_k * split / p.splits), t1 = (int)((int64_t)tiles_k * (split + 1) / p.splits);

  const uint16_t* const kbase = p.k + s.b * p.kb + s.k0 * p.kt + kv_head * p.kh;
  const uint16_t* const vbase = p.v + s.b * p.vb + s.k0 * p.vt + kv_head * p.vh;
  // DMA i of this wave: 1 KB of the tile's rows.
  uint32_t koff[DMAS], voff[DMAS];
#pragma unroll
  for (int i = 0; i < DMAS; ++i) {
    const int at = (wave * DMAS + i) * 64 + lane;  // 16-byte slot of the tile
    const int row = at / CH, c = at % CH ^ (row / RPB % PAIRS) * 2;
    koff[i] = (uint32_t)(row * p.kt * 2 + c * 16);
    voff[i] = (uint32_t)(row * p.vt * 2 + c * 16);
  }
  auto issue = [&](int t) {
    if (t >= t1) return;
    char* const slot = smem + t % S * SLOT;
    const int left = min(kKeys, s.kn - t * kKeys);  // rows past the sequence's keys read as zero
    const __amdgpu_buffer_rsrc_t rk =
        row_rsrc(kbase + (int64_t)t * kKeys * p.kt, ((int64_t)(left - 1) * p.kt + D) * 2);
    const __amdgpu_buffer_rsrc_t rv =
        row_rsrc(vbase + (int64_t)t * kKeys * p.vt, ((int64_t)(left - 1) * p.vt + D) * 2);
#pragma unroll
    for (int i = 0; i < DMAS; ++i)
      dma16(rk, slot + (wave * DMAS + i) * 1024, koff[i]);
#pragma unroll
    for (int i = 0; i < DMAS; ++i)
      dma16(rv, slot + TILE + (wave * DMAS + i) * 1024, voff[i]);
  };

  v16f o[QB][DB];
  float m[QB], l[QB];
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    m[b] = -INFINITY;
    l[b] = 0.0f;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[b][d][e] = 0.0f;
  }

  issue(t0);
#pragma unroll 1
  for (int t = t0; t < t1; ++t) {
    __builtin_amdgcn_s_waitcnt(0x70 | 0xf00);  // vmcnt(0): tile t has landed
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    issue(t + 1);  // into the slot that every wave left before the barrier
    const char* const ks = smem + t % S * SLOT;
    const char* const vs = ks + TILE;
    v16f sc[QB][2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int b = 0; b < QB; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[b][kb][e] = 0.0f;
#pragma unroll
      for (int d = 0; d < KD; ++d) {
        const int row = 32 * kb + col;
        const V8 kf = *reinterpret_cast<const V8*>(ks + row * ROW +
                                                   ((2 * d + half) ^ (row / RPB % PAIRS) * 2) * 16);
#pragma unroll
        for (int b = 0; b < QB; ++b) sc[b][kb] = Mfma<T>::mul(kf, q[b][d], sc[b][kb]);
      }
    }
    if ((t + 1) * kKeys > sure) {
#pragma unroll
      for (int b = 0; b < QB; ++b)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = t * kKeys + 32 * kb + 8 * (e >> 2) + 4 * half + (e & 3);
            sc[b][kb][e] = key < limit[b] ? sc[b][kb][e] : -INFINITY;
          }
    }
    uint32_t pk[QB][2][8];
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      float mx = fmaxf(sc[b][0][0], sc[b][1][0]);
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, fmaxf(sc[b][0][e], sc[b][1][e]));
      mx = max_with_partner(mx);
      if (__any((mx - m[b]) * p.c > kSlack || (m[b] == -INFINITY && mx > -INFINITY))) {
        const float mn = fmaxf(m[b], mx);
        const float alpha = m[b] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[b] - mn) * p.c);
        m[b] = mn;
        l[b] *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[b][d][e] *= alpha;
      }
      const float off = m[b] == -INFINITY ? 0.0f : m[b] * p.c - kShift;
      float sum = 0.0f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][kb][e], p.c, -off));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][kb][e + 1], p.c, -off));
          sum += p0 + p1;
          pk[b][kb][e >> 1] = Mfma<T>::pack(p0, p1);
        }
      l[b] += sum;
    }
#pragma unroll
    for (int kc = 0; kc < 4; ++kc) {  // 16 keys
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        // Lane's column 32 * d + col; its keys 16 * kc + 4 * half + (0..3, 8..11).
        const int i16 = lane & 15;
        const int row = 16 * kc + 4 * half + (i16 >> 2);
        const int c = 4 * d + 2 * ((lane >> 4) & 1) + (i16 >> 1 & 1);
        const int sub = (i16 & 1) * 8;
        const char* const a0 = vs + row * ROW + (c ^ (row / RPB % PAIRS) * 2) * 16 + sub;
        const char* const a1 = vs + (row + 8) * ROW + (c ^ ((row + 8) / RPB % PAIRS) * 2) * 16 + sub;
        const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t)a0);
        const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t)a1);
        const V8 vf = __builtin_bit_cast(V8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int b = 0; b < QB; ++b) {
          const uint4 pw = make_uint4(pk[b][kc >> 1][(kc & 1) * 4], pk[b][kc >> 1][(kc & 1) * 4 + 1],
                                      pk[b][kc >> 1][(kc & 1) * 4 + 2], pk[b][kc >> 1][(kc & 1) * 4 + 3]);
          o[b][d] = Mfma<T>::mul(vf, __builtin_bit_cast(V8, pw), o[b][d]);
        }
      }
    }
  }

  // o / l; lane holds columns 32 * d + 8 * g + 4 * half + 0..3 of its row.
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const int64_t r = r0 + wave * 32 * QB + 32 * b + col;
    const float sum = add_partner(l[b]);
    if (r >= rows) continue;
    const int64_t row = (s.b * p.q_rows + s.q0 + tok[b]) * p.heads + head[b];
    if (p.splits > 1) {
      const int64_t all = (p.cu_q ? 1 : p.n) * p.q_rows * p.heads;
      float* const po = p.part + (split * all + row) * D;
      float* const ml = p.part + (int64_t)p.splits * all * D + (split * all + row) * 2;
      if (half == 0) {
        ml[0] = m[b];
        ml[1] = sum;
      }
      // A split without keys of this row is left out of the sum by its l of 0.
      if (sum != 0.0f) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4*>(po + 32 * d + 8 * g + 4 * half) =
                make_float4(o[b][d][4 * g], o[b][d][4 * g + 1], o[b][d][4 * g + 2], o[b][d][4 * g + 3]);
      }
      continue;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t* const po = p.out + row * D;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<uint2*>(po + 32 * d + 8 * g + 4 * half) =
            make_uint2(Mfma<T>::pack(o[b][d][4 * g] * inv, o[b][d][4 * g + 1] * inv),
                       Mfma<T>::pack(o[b][d][4 * g + 2] * inv, o[b][d][4 * g + 3] * inv));
  }
}

// Joins the splits of a row: weights 2^(c (m_s - max m)), in split order.
template <typename T, int D>
__global__ __launch_bounds__(256) void join_splits(const float* __restrict__ part, uint16_t* __restrict__ out,
                                                   int64_t rows, int splits, float c) {
  constexpr int LANES = D / 4;  // threads of a row, four columns each
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES;
  const int at = threadIdx.x % LANES * 4;
  if (row >= rows) return;
  const float* const ml = part + (int64_t)splits * rows * D;
  float m = -INFINITY;
  for (int s = 0; s < splits; ++s) {
    const float2 v = *reinterpret_cast<const float2*>(ml + (s * rows + row) * 2);
    if (v.y != 0.0f) m = fmaxf(m, v.x);
  }
  float l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < splits; ++s) {
    const float2 v = *reinterpret_cast<const float2*>(ml + (s * rows + row) * 2);
    if (v.y == 0.0f) continue;
    const float w = __builtin_amdgcn_exp2f((v.x - m) * c);
    const float4 x = *reinterpret_cast<const float4*>(part + (s * rows + row) * D + at);
    l += w * v.y;
    o[0] += w * x.x;
    o[1] += w * x.y;
    o[2] += w * x.z;
    o[3] += w * x.w;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<uint2*>(out + row * D + at) =
      make_uint2(Mfma<T>::pack(o[0] * inv, o[1] * inv), Mfma<T>::pack(o[2] * inv, o[3] * inv));
}

// How a call is laid over the GPU.
struct Plan {
  int pack, rows, splits;  // query heads per tile row space, rows per tile
  int64_t tiles;           // row tiles per head in all
};

Plan plan(int64_t n, int64_t q_rows, int64_t k_rows, bool packed, int heads, int kv_heads) {
  const int group = heads / kv_heads;
  const int64_t mean_q = packed ? (n > 0 ? q_rows / n : 0) : q_rows;   // rows per sequence
  const int64_t mean_k = packed ? (n > 0 ? k_rows / n : 0) : k_rows;
  Plan pl;
  const bool few = mean_q * group <= 64;
  pl.pack = few ? group : 1;
  pl.rows = few && mean_q * group <= 32 ? 32 : 128;
  const int64_t slots = kMaxBlocks;
  pl.tiles = packed ? q_rows * pl.pack / pl.rows + n + 2
                    : n * ((q_rows * pl.pack + pl.rows - 1) / pl.rows);
  const int64_t work = pl.tiles * (heads / pl.pack);
  const int64_t want = pl.rows == 32 ? 4 * compute_units() : compute_units();
  int64_t s = work > 0 ? want / work : 1;
  const int64_t most = mean_k / 256;   // at least 256 keys each
  s = s < most ? s : most;
  pl.splits = (int)(s < 1 ? 1 : (s > 256 ? 256 : s));
  while (pl.splits > 1 && work * pl.splits > slots) --pl.splits;
  return pl;
}

template <typename T, int D>
int launch(AttnArgs p, const Plan& pl, hipStream_t s) {
  const int64_t grid = pl.tiles * (p.heads / pl.pack) * pl.splits;
  LR_REQUIRE(grid <= kMaxBlocks, "attention: %lld workgroups are not supported", (long long)grid);
  if (pl.rows == 32) attention<T, D, 1, 1, 2><<<(unsigned)grid, 64, 0, s>>>(p);
  else attention<T, D, 1, 4, 2><<<(unsigned)grid, 256, 0, s>>>(p);
  if (int rc = check_launch("attention")) return rc;
  if (pl.splits == 1) return LR_OK;
  const int64_t rows = (p.cu_q ? 1 : p.n) * p.q_rows * p.heads, blocks = (rows * (D / 4) + 255) / 256;
  LR_REQUIRE(blocks <= kMaxBlocks, "attention: %lld rows are not supported", (long long)rows);
  join_splits<T, D><<<(unsigned)blocks, 256, 0, s>>>(p.part, p.out, rows, pl.splits, p.c);
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

extern "C" int lr_attention_splits(int64_t sequences, int64_t q_rows, int64_t k_rows, int packed, int heads,
                                   int kv_heads) {
  if (sequences <= 0 || q_rows <= 0 || k_rows <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return 1;
  return plan(sequences, q_rows, k_rows, packed != 0, heads, kv_heads).splits;
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
  LR_REQUIRE(splits >= 1 && splits <= 256, "attention: %d splits", splits);
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
  Plan pl = plan(sequences, q_rows, k_rows, packed, heads, kv_heads);
  pl.splits = splits;
  p.pack = pl.pack;
  p.tiles = pl.tiles;
  p.splits = splits;
  if (splits > 1) {
    const int64_t rows = (packed ? 1 : sequences) * q_rows * heads;
    LR_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= splits * rows * (head_dim + 2) * 4,
               "attention: %d splits need a workspace of %lld bytes", splits,
               (long long)(splits * rows * (head_dim + 2) * 4));
  }
  hipStream_t s = as_stream(stream);
  return dtype == LR_DTYPE_BF16 ? by_dim<__bf16>(p, head_dim, pl, s) : by_dim<_Float16>(p, head_dim, pl, s);
}
