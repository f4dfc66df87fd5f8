// adapters.hip - low-rank adapters of many requests beside a shared projection:
//
//   out[t] = base[t] + scale[a] (x[t] down[a]^T) up[a]^T,   a = index[t], or base[t] without one
//
// with down[a] [rank, k] and up[a] [n, rank]. A plan, made once for a batch and used by
// every layer, lists the tokens by adapter in tiles of at most 64. Two kernels:
//   shrink   inner[t] = x[t] down[a]^T, fp32, a tile of tokens and a share of k per workgroup
//   expand   adds up a token's shares in order, scales them, and adds the product with up
//            to the projection, a tile of tokens and a run of columns per workgroup
// Both are bound by memory: x, base and out pass once, an adapter once per tile of tokens
// (out of the L2 from the second on). inner goes to the second product as two 16-bit numbers,
// rounded and rest, of a row scaled by a power of two, so that only out is rounded in the end.
#include "lr_attention.h"
#include "lr_runtime.h"

namespace lr {
namespace {

constexpr int kTokens = 64;         // of a tile
constexpr int kMaxAdapters = 1000;  // a plan counts each wave's tokens of them in 64 KB of LDS
constexpr int kMaxRank = 128;
constexpr int kStep = 64;           // columns of x per step of shrink
constexpr int kColumns = 128;       // columns of out per step of expand
// An offset past every buffer here: such a lane reads zeros.
constexpr uint32_t kOutside = 0xfff80000u;
constexpr int64_t kMaxWindow = 0xfff00000ll;

// Tiles that a plan may have: full ones, and one more for each adapter in use.
int64_t plan_tiles(int64_t tokens, int64_t adapters) {
  return tokens / kTokens + (adapters + 1 < tokens ? adapters + 1 : tokens);
}

// -------------------------------------------------------------------- plan ----
constexpr int kPlan = 1024;   // threads

// A counting sort by one workgroup: every wave counts its stretch of the tokens, then puts
// them in their places in order. Tokens without an adapter (an index outside 0 .. adapters - 1)
// come last, as those of adapter -1.
__global__ __launch_bounds__(kPlan) void plan_adapters(const int32_t* index, int tokens, int adapters, int32_t* order,
                                                       int4* tiles, int max_tiles) {
  constexpr int WAVES = kPlan / 64;
  extern __shared__ int counts[];   // [WAVES][adapters + 1]: tokens, then their next place
  __shared__ int sums[2][WAVES];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, kinds = adapters + 1;
  for (int i = t; i < WAVES * kinds; i += kPlan) counts[i] = 0;
  __syncthreads();
  auto kind_of = [&](int i) __attribute__((always_inline)) {
    const int a = index[i];
    return (uint32_t)a < (uint32_t)adapters ? a : adapters;
  };
  int* const mine = counts + wave * kinds;
  const int stretch = ((tokens + WAVES - 1) / WAVES + 63) & ~63;
  const int i0 = min(tokens, wave * stretch), i1 = min(tokens, i0 + stretch);
  for (int i = i0 + lane; i < i1; i += 64) atomicAdd(&mine[kind_of(i)], 1);
  __syncthreads();
  // Thread t has kinds 2 t and 2 t + 1: their tokens and tiles, and those before them.
  int n[2] = {0, 0}, need[2];
  for (int j = 0; j < 2; ++j) {
    const int a = 2 * t + j;
    if (a < kinds)
      for (int w = 0; w < WAVES; ++w) n[j] += counts[w * kinds + a];
    need[j] = (n[j] + kTokens - 1) / kTokens;
  }
  const int upto_n = wave_prefix_sum(n[0] + n[1]), upto_t = wave_prefix_sum(need[0] + need[1]);
  if (lane == 63) {
    sums[0][wave] = upto_n;
    sums[1][wave] = upto_t;
  }
  __syncthreads();
  int place = upto_n - n[0] - n[1], tile = upto_t - need[0] - need[1], all = 0;
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) {
      place += sums[0][w];
      tile += sums[1][w];
    }
    all += sums[1][w];
  }
  for (int j = 0; j < 2; ++j) {
    const int a = 2 * t + j;
    if (a >= kinds) break;
    int at = place;
    for (int w = 0; w < WAVES; ++w) {   // the waves' first places, in their order
      const int c = counts[w * kinds + a];
      counts[w * kinds + a] = at;
      at += c;
    }
    for (int i = 0; i < need[j]; ++i)
      tiles[tile + i] = make_int4(a < adapters ? a : -1, place + i * kTokens, min(kTokens, n[j] - i * kTokens), 0);
    place += n[j];
    tile += need[j];
  }
  for (int i = all + t; i < max_tiles; i += kPlan) tiles[i] = make_int4(-1, 0, 0, 0);
  __syncthreads();
  for (int i = i0; i < i1; i += 64) {
    const int at = i + lane, a = at < i1 ? kind_of(at) : -1;
    uint64_t left = __ballot(at < i1);
    while (left) {   // the tokens of one adapter after the other
      const int one = __builtin_amdgcn_readlane(a, __builtin_ctzll(left));
      const uint64_t same = __ballot(a == one);
      if (a == one) order[mine[one] + __builtin_popcountll(same & ((1ULL << lane) - 1))] = at;
      if (a == one && (same & ((1ULL << lane) - 1)) == 0) mine[one] += __builtin_popcountll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the next read of it is another lane's
      left &= ~same;
    }
  }
}

// ------------------------------------------------------------------ shrink ----
struct AdapterArgs {
  const uint16_t *x, *down, *up, *base;
  const float* scale;
  uint16_t* out;
  float* part;           // shares of inner [splits][tiles][64][padded rank]
  const int32_t* order;
  const int4* tiles;
  int64_t xs, bs, os;    // row strides in elements
  int64_t first;         // token of this window of x, and how many: what 32-bit offsets reach
  int window;
  int tokens, n, k, rank, max_tiles;
  int k8, rank8;         // rows of down and up, in elements
  int splits;            // of k
  int columns;           // of a workgroup of expand
  int vector;            // whether base and out are read and written 16 bytes at a time
};

template <int COUNT>
__device__ __forceinline__ void wait_loads() {   // all but the last COUNT
  static_assert(COUNT < 64, "vmcnt");
  __builtin_amdgcn_s_waitcnt((COUNT & 15) | (COUNT >> 4) << 14 | 0x70 | 0xf00);
}

// Four waves; steps of 64 columns through a ring of LDS slots that hold 64 rows of x and RP of
// down, 128 bytes each (16-byte chunk c of row r in place c ^ r % 8). Wave w takes the columns
// 16 w .. of a step for all rows, so that each element leaves the LDS once; the waves' sums are
// added at the end. The product is transposed, down x^T: a lane holds four ranks of a token
// next to each other.
template <typename T, int RP>
__global__ __launch_bounds__(256) void shrink(AdapterArgs p) {
  typedef typename Mfma<T>::V V8;
  constexpr int RB = RP / 32, TB = kTokens / 32, ROW = 2 * kStep, RING = 4;
  constexpr int SLOT = (kTokens + RP) * ROW, XD = kTokens / 8 / 4, DD = RP / 8 / 4;   // DMAs of a wave
  constexpr int GROUP = 4 < TB * RB ? 4 : TB * RB;   // blocks that are added at a time
  static_assert(RING * SLOT >= 4 * GROUP * 4096, "the sums take the ring's place");
  __shared__ __attribute__((aligned(1024))) char smem[RING * SLOT];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int half = lane >> 5, col = lane & 31;
  const int tile = (int)(blockIdx.x % (uint32_t)p.max_tiles), split = (int)(blockIdx.x / (uint32_t)p.max_tiles);
  const int4 info = p.tiles[tile];
  const int a = info.x, count = info.z;
  if (a < 0 || count == 0) return;
  const int steps = (p.k + kStep - 1) / kStep, chunk = (steps + p.splits - 1) / p.splits;
  const int s0 = min(steps, split * chunk), s1 = min(steps, s0 + chunk);
  const __amdgpu_buffer_rsrc_t xr = row_rsrc(p.x + p.first * p.xs, ((int64_t)(p.window - 1) * p.xs + p.k8) * 2);
  const __amdgpu_buffer_rsrc_t dr = row_rsrc(p.down + (int64_t)a * p.rank * p.k8, (int64_t)p.rank * p.k8 * 2);
  // This lane's rows and chunk of each DMA (8 rows of 128 bytes).
  uint32_t xo[XD], dof[DD];
  int mine = 0;   // rows of this window
  const int at = (lane & 7) ^ (lane >> 3);   // chunk of a step (rows of a DMA start at multiples of 8)
#pragma unroll
  for (int i = 0; i < XD; ++i) {
    const int r = (wave * XD + i) * 8 + (lane >> 3);
    const int64_t tok = r < count ? p.order[info.y + r] - p.first : -1;
    const bool in = tok >= 0 && tok < p.window;
    xo[i] = in ? (uint32_t)(tok * p.xs * 2 + at * 16) : kOutside;
    mine += in;
  }
  if (__syncthreads_count(mine) == 0) return;
#pragma unroll
  for (int i = 0; i < DD; ++i) {
    const int r = (wave * DD + i) * 8 + (lane >> 3);
    dof[i] = r < p.rank ? (uint32_t)((int64_t)r * p.k8 * 2 + at * 16) : kOutside;
  }
  auto issue = [&](int s) {
    char* const slot = smem + (s - s0) % RING * SLOT;
    // Chunks past the last column read as zero on both sides.
    const bool in = s < s1 && s * kStep + at * 8 < p.k8;
    const uint32_t off = (uint32_t)s * (kStep * 2);
#pragma unroll
    for (int i = 0; i < XD; ++i)
      dma16(xr, slot + (wave * XD + i) * 1024, in && xo[i] != kOutside ? xo[i] + off : kOutside);
#pragma unroll
    for (int i = 0; i < DD; ++i)
      dma16(dr, slot + kTokens * ROW + (wave * DD + i) * 1024, in && dof[i] != kOutside ? dof[i] + off : kOutside);
  };
  v16f acc[TB][RB];
#pragma unroll
  for (int b = 0; b < TB; ++b)
#pragma unroll
    for (int c = 0; c < RB; ++c)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[b][c][e] = 0.0f;
  const int place = ((2 * wave + half) ^ (col & 7)) * 16;
#pragma unroll
  for (int i = 0; i < RING - 1; ++i) issue(s0 + i);
#pragma unroll 1
  for (int s = s0; s < s1; ++s) {
    wait_loads<(RING - 2) * (XD + DD)>();
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();   // step s is there, and every wave is done with step s - 1
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    issue(s + RING - 1);
    const char* const slot = smem + (s - s0) % RING * SLOT;
    V8 df[RB];
#pragma unroll
    for (int c = 0; c < RB; ++c) df[c] = *reinterpret_cast<const V8*>(slot + (kTokens + 32 * c + col) * ROW + place);
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      if (32 * b >= count) continue;
      const V8 xf = *reinterpret_cast<const V8*>(slot + (32 * b + col) * ROW + place);
#pragma unroll
      for (int c = 0; c < RB; ++c) acc[b][c] = Mfma<T>::mul(df[c], xf, acc[b][c]);
    }
  }
  float4* const sums = reinterpret_cast<float4*>(smem);
  float* const part = p.part + ((int64_t)split * p.max_tiles + tile) * kTokens * RP;
#pragma unroll
  for (int g0 = 0; g0 < TB * RB; g0 += GROUP) {
    wait_loads<0>();
    __syncthreads();   // nothing is on its way to the ring, and what is read of it has been
#pragma unroll
    for (int g = 0; g < GROUP; ++g)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const v16f& v = acc[(g0 + g) / RB][(g0 + g) % RB];
        sums[((wave * GROUP + g) * 4 + q) * 64 + lane] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
      }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < GROUP; ++g) {
      // Thread: quarter `wave` of block g0 + g.
      float4 v = sums[(g * 4 + wave) * 64 + lane];
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        const float4 y = sums[((w * GROUP + g) * 4 + wave) * 64 + lane];
        v.x += y.x;
        v.y += y.y;
        v.z += y.z;
        v.w += y.w;
      }
      const int tok = (g0 + g) / RB * 32 + col, r = (g0 + g) % RB * 32 + 8 * wave + 4 * half;
      if (tok >= count) continue;
      if (p.window < p.tokens) {   // rows of other windows are theirs to write
        const int64_t of = p.order[info.y + tok] - p.first;
        if (of < 0 || of >= p.window) continue;
      }
      *reinterpret_cast<float4*>(part + tok * RP + r) = v;
    }
  }
}

// ------------------------------------------------------------------ expand ----
template <typename T> __device__ __forceinline__ float to_float(uint16_t v) {
  return (float)__builtin_bit_cast(T, v);
}

// Four waves: 32 tokens x 64 columns each of a step of 128 columns. up's rows come through
// LDS like the keys of lr_attention.h (a row holds RP numbers); the sums leave through LDS
// too, so that base and out are read and written in whole lines.
template <typename T, int RP>
__global__ __launch_bounds__(256) void expand(AdapterArgs p) {
  typedef typename Mfma<T>::V V8;
  constexpr int ROW = 2 * RP, CH = ROW / 16, RPB = 256 / ROW, PAIRS = ROW / 32, KR = RP / 16;
  constexpr int UP = kColumns * ROW, DMAS = UP / 1024 / 4, PITCH = kColumns + 4;
  constexpr int INNER = 2 * kTokens * ROW;   // rounded and rest
  constexpr int OUT = kTokens * PITCH * 4;
  __shared__ __attribute__((aligned(1024))) char smem[UP + (OUT > INNER ? OUT : INNER)];
  __shared__ float exponents[kTokens];
  __shared__ int tokens[kTokens];
  char* const inner = smem + UP;
  float* const result = reinterpret_cast<float*>(smem + UP);
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const int half = lane >> 5, col = lane & 31;
  const int tile = (int)(blockIdx.x % (uint32_t)p.max_tiles), run = (int)(blockIdx.x / (uint32_t)p.max_tiles);
  const int4 info = p.tiles[tile];
  const int a = info.x, count = info.z;
  if (count == 0 || (a < 0 && p.out == p.base)) return;
  const int n0 = run * p.columns, n1 = min(p.n, n0 + p.columns);
  if (t < kTokens) tokens[t] = t < count ? p.order[info.y + t] : 0;
  // Step c: this thread's row (16 threads of 8 columns each, 16 rows at a time) of base.
  const int c8 = (t & 15) * 8, row0 = t >> 4;
  uint4 kept[kTokens / 16];
  auto load_base = [&](int c) {
#pragma unroll
    for (int i = 0; i < kTokens / 16; ++i) {
      const int r = 16 * i + row0, n = c + c8;
      if (r >= count || n >= n1) continue;
      const uint16_t* const from = p.base + tokens[r] * p.bs + n;
      if (p.vector) kept[i] = load_nt(reinterpret_cast<const uint4*>(from));
      else
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          set_word(kept[i], e / 2, (n + e < n1 ? from[e] : 0u) | (n + e + 1 < n1 ? (uint32_t)from[e + 1] << 16 : 0u));
    }
  };
  auto store_out = [&](int c) {
#pragma unroll
    for (int i = 0; i < kTokens / 16; ++i) {
      const int r = 16 * i + row0, n = c + c8;
      if (r >= count || n >= n1) continue;
      uint16_t* const to = p.out + tokens[r] * p.os + n;
      if (p.vector) store_nt(reinterpret_cast<uint4*>(to), kept[i]);
      else
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < n1) to[e] = (uint16_t)(word(kept[i], e / 2) >> (16 * (e & 1)));
    }
  };
  __syncthreads();
  if (a < 0) {
    for (int c = n0; c < n1; c += kColumns) {
      load_base(c);
      store_out(c);
    }
    return;
  }
  const uint16_t* const up = p.up + (int64_t)a * p.n * p.rank8;
  auto issue = [&](int c) {
    const __amdgpu_buffer_rsrc_t r = row_rsrc(up + (int64_t)c * p.rank8, (int64_t)min(kColumns, p.n - c) * p.rank8 * 2);
#pragma unroll
    for (int i = 0; i < DMAS; ++i) {
      const int s = (wave * DMAS + i) * 64 + lane, row = s / CH, ch = s % CH ^ (row / RPB % PAIRS) * 2;
      dma16(r, smem + (wave * DMAS + i) * 1024, ch * 8 < p.rank8 ? (uint32_t)(row * p.rank8 * 2 + ch * 16) : kOutside);
    }
  };
  issue(n0);
  load_base(n0);
  {
    // inner of the tile: four threads a token, RP / 4 ranks each.
    constexpr int EACH = RP / 4;
    const int tok = t >> 2, r0 = (t & 3) * EACH;
    float v[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) v[e] = 0.0f;
    if (tok < count) {
      const float* from = p.part + ((int64_t)tile * kTokens + tok) * RP + r0;
      for (int s = 0; s < p.splits; ++s, from += (int64_t)p.max_tiles * kTokens * RP)
#pragma unroll
        for (int e = 0; e < EACH; e += 4) {
          const float4 y = *reinterpret_cast<const float4*>(from + e);
          v[e] += y.x;
          v[e + 1] += y.y;
          v[e + 2] += y.z;
          v[e + 3] += y.w;
        }
    }
    const float scale = p.scale[a];
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      v[e] = r0 + e < p.rank ? v[e] * scale : 0.0f;   // (a row past the rank may hold 0 * infinity)
      top = fmaxf(top, __builtin_fabsf(v[e]));
    }
    top = fmaxf(top, xor_partner<1>(top));
    top = fmaxf(top, xor_partner<2>(top));
    // The largest of the row to [1, 2); what is infinite or zero stays.
    const int ex = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 1 : 0;
    if ((t & 3) == 0) exponents[tok] = __builtin_amdgcn_ldexpf(1.0f, ex);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; e += 8) {
      uint4 hi, lo;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y0 = __builtin_amdgcn_ldexpf(v[e + 2 * j], -ex), y1 = __builtin_amdgcn_ldexpf(v[e + 2 * j + 1], -ex);
        const uint32_t w = Mfma<T>::pack(y0, y1);
        const float d0 = y0 - Mfma<T>::first(w), d1 = y1 - Mfma<T>::second(w);
        set_word(hi, j, w);
        // An infinity has no rest.
        set_word(lo, j, Mfma<T>::pack(__builtin_fabsf(y0) < INFINITY ? d0 : 0.0f, __builtin_fabsf(y1) < INFINITY ? d1 : 0.0f));
      }
      const int ch = (r0 + e) / 8 ^ (tok / RPB % PAIRS) * 2;
      *reinterpret_cast<uint4*>(inner + tok * ROW + ch * 16) = hi;
      *reinterpret_cast<uint4*>(inner + kTokens * ROW + tok * ROW + ch * 16) = lo;
    }
    __syncthreads();
  }
  const int row = 32 * (wave & 1) + col, first = 64 * (wave >> 1);   // the lane's token, the wave's columns of a step
  const bool idle = 32 * (wave & 1) >= count;
  V8 hi[KR], lo[KR];
#pragma unroll
  for (int d = 0; d < KR; ++d) {
    const int ch = (2 * d + half) ^ (row / RPB % PAIRS) * 2;
    hi[d] = *reinterpret_cast<const V8*>(inner + row * ROW + ch * 16);
    lo[d] = *reinterpret_cast<const V8*>(inner + kTokens * ROW + row * ROW + ch * 16);
  }
  const float back = exponents[row];
  for (int c = n0; c < n1; c += kColumns) {
    wait_loads<0>();
    __syncthreads();   // up's rows are there; inner, or the step before, has been read
    if (!idle) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        v16f s;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.0f;
        const int n = first + 32 * b + col;
#pragma unroll
        for (int d = 0; d < KR; ++d) {
          const V8 uf = *reinterpret_cast<const V8*>(smem + n * ROW + ((2 * d + half) ^ (n / RPB % PAIRS) * 2) * 16);
          s = Mfma<T>::mul(uf, lo[d], s);
          s = Mfma<T>::mul(uf, hi[d], s);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4*>(result + row * PITCH + first + 32 * b + 8 * g + 4 * half) =
              make_float4(s[4 * g] * back, s[4 * g + 1] * back, s[4 * g + 2] * back, s[4 * g + 3] * back);
      }
    }
    __syncthreads();
    if (c + kColumns < n1) issue(c + kColumns);
#pragma unroll
    for (int i = 0; i < kTokens / 16; ++i) {
      const int r = 16 * i + row0;
      if (r >= count) continue;
      const float4 y0 = *reinterpret_cast<const float4*>(result + r * PITCH + c8);
      const float4 y1 = *reinterpret_cast<const float4*>(result + r * PITCH + c8 + 4);
      const float y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t w = word(kept[i], e);
        set_word(kept[i], e, Mfma<T>::pack(Mfma<T>::first(w) + y[2 * e], Mfma<T>::second(w) + y[2 * e + 1]));
      }
    }
    store_out(c);
    if (c + kColumns < n1) load_base(c + kColumns);
  }
}

struct AddPlan {
  int rank;      // padded
  int splits, columns;
  int64_t tiles, bytes;
};

AddPlan add_plan(int64_t tokens, int64_t n, int64_t k, int rank, int64_t adapters) {
  AddPlan pl;
  pl.rank = rank <= 32 ? 32 : (rank <= 64 ? 64 : 128);
  pl.tiles = plan_tiles(tokens, adapters);
  const int64_t want = 2 * compute_units(), steps = (k + kStep - 1) / kStep;
  // Shares of k of at least four steps, at most 16 of them, to two workgroups per CU.
  int64_t s = (want + pl.tiles - 1) / pl.tiles;
  if (s > steps / 4) s = steps / 4;
  pl.splits = s < 1 ? 1 : (s > 16 ? 16 : (int)s);
  // Columns of an expanding workgroup: up to 1024, less where that leaves CUs idle.
  int64_t c = 1024;
  while (c > kColumns && pl.tiles * ((n + c - 1) / c) < want) c /= 2;
  pl.columns = (int)c;
  pl.bytes = pl.splits * pl.tiles * kTokens * pl.rank * 4;
  return pl;
}

template <typename T, int RP>
int add(AdapterArgs p, const AddPlan& pl, hipStream_t s) {
  const int64_t rows = kMaxWindow / (p.xs * 2 > 2 * p.k8 ? p.xs * 2 : 2 * p.k8);
  for (int64_t first = 0; first < p.tokens; first += rows) {
    p.first = first;
    p.window = (int)(p.tokens - first < rows ? p.tokens - first : rows);
    shrink<T, RP><<<(unsigned)(pl.tiles * pl.splits), 256, 0, s>>>(p);
    if (int rc = check_launch("adapter_add")) return rc;
  }
  expand<T, RP><<<(unsigned)(pl.tiles * ((p.n + pl.columns - 1) / pl.columns)), 256, 0, s>>>(p);
  return check_launch("adapter_add");
}

template <typename T>
int add_by_rank(const AdapterArgs& p, const AddPlan& pl, hipStream_t s) {
  if (pl.rank == 32) return add<T, 32>(p, pl, s);
  if (pl.rank == 64) return add<T, 64>(p, pl, s);
  return add<T, 128>(p, pl, s);
}

int check_add(int64_t tokens, int64_t n, int64_t k, int rank, int64_t adapters) {
  LR_REQUIRE(tokens >= 0 && n > 0 && k > 0 && rank > 0 && adapters > 0, "adapter_add: negative or empty shape");
  if (rank > kMaxRank) return fail(LR_EUNSUPPORTED, "adapter_add: rank %d is not supported (at most %d)", rank, kMaxRank);
  if (adapters > kMaxAdapters)
    return fail(LR_EUNSUPPORTED, "adapter_add: %lld adapters are not supported (at most %d)", (long long)adapters, kMaxAdapters);
  LR_REQUIRE(tokens < (1LL << 24) && n < (1LL << 24) && k <= (1LL << 23),
             "adapter_add: 2^24 tokens or outputs, or more than 2^23 inputs, are not supported");
  return LR_OK;
}

}  // namespace
}  // namespace lr

using namespace lr;

extern "C" int lr_adapter_tiles(int64_t tokens, int adapters) {
  return tokens > 0 && tokens < (1LL << 24) && adapters > 0 && adapters <= kMaxAdapters ? (int)plan_tiles(tokens, adapters) : 0;
}

extern "C" int lr_adapter_plan(const int32_t* index, int64_t tokens, int adapters, int32_t* order, int32_t* tiles, void* stream) {
  if (int rc = check_add(tokens, 1, 1, 1, adapters)) return rc;
  if (tokens == 0) return LR_OK;
  LR_REQUIRE(index && order && tiles, "adapter_plan: null pointer");
  LR_REQUIRE(aligned(index, 4) && aligned(order, 4) && aligned(tiles, 16), "adapter_plan: tiles must be 16-byte aligned");
  const int lds = kPlan / 64 * (adapters + 1) * 4;
  plan_adapters<<<1, kPlan, lds, as_stream(stream)>>>(index, (int)tokens, adapters, order, reinterpret_cast<int4*>(tiles),
                                                     (int)plan_tiles(tokens, adapters));
  return check_launch("adapter_plan");
}

extern "C" int lr_adapter_workspace(int64_t tokens, int64_t n, int64_t k, int rank, int adapters, int64_t* bytes) {
  if (int rc = check_add(tokens, n, k, rank, adapters)) return rc;
  LR_REQUIRE(bytes, "adapter_add: null pointer");
  *bytes = tokens ? add_plan(tokens, n, k, rank, adapters).bytes : 0;
  return LR_OK;
}

extern "C" int lr_adapter_add(const void* x, int64_t x_stride, const void* down, const void* up, const float* scale,
                              const void* base, int64_t base_stride, void* out, int64_t out_stride, int dtype,
                              int64_t tokens, int64_t n, int64_t k, int rank, int adapters, const int32_t* order,
                              const int32_t* tiles, void* workspace, int64_t workspace_bytes, void* stream) {
  LR_REQUIRE(dtype == LR_DTYPE_BF16 || dtype == LR_DTYPE_F16, "adapter_add: unknown dtype %d", dtype);
  if (int rc = check_add(tokens, n, k, rank, adapters)) return rc;
  if (tokens == 0) return LR_OK;
  LR_REQUIRE(x && down && up && scale && base && out && order && tiles, "adapter_add: null pointer");
  LR_REQUIRE(aligned(x, 16) && aligned(down, 16) && aligned(up, 16) && aligned(scale, 4) && aligned(order, 4) &&
                 aligned(tiles, 16) && aligned(base, 2) && aligned(out, 2),
             "adapter_add: inputs and adapters must be 16-byte aligned");
  const int64_t k8 = (k + 7) & ~7LL;
  LR_REQUIRE(x_stride >= 0 && x_stride % 8 == 0 && (x_stride >= k8 || tokens == 1 || x_stride == 0),
             "adapter_add: rows of x %lld elements apart, not a multiple of 8 of at least %lld", (long long)x_stride,
             (long long)k8);
  LR_REQUIRE(x_stride < (1LL << 30) && base_stride >= 0 && (out_stride >= n || tokens == 1),
             "adapter_add: rows of %lld columns %lld apart", (long long)n, (long long)out_stride);
  const AddPlan pl = add_plan(tokens, n, k, rank, adapters);
  const int64_t runs = (n + pl.columns - 1) / pl.columns;
  LR_REQUIRE(pl.tiles * pl.splits <= kMaxBlocks && pl.tiles * runs <= kMaxBlocks,
             "adapter_add: %lld tiles of tokens are not supported", (long long)pl.tiles);
  LR_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= pl.bytes,
             "adapter_add: needs a workspace of %lld bytes", (long long)pl.bytes);
  AdapterArgs p = {};
  p.x = static_cast<const uint16_t*>(x);
  p.down = static_cast<const uint16_t*>(down);
  p.up = static_cast<const uint16_t*>(up);
  p.base = static_cast<const uint16_t*>(base);
  p.scale = scale;
  p.out = static_cast<uint16_t*>(out);
  p.part = static_cast<float*>(workspace);
  p.order = order;
  p.tiles = reinterpret_cast<const int4*>(tiles);
  p.xs = x_stride;
  p.bs = base_stride;
  p.os = out_stride;
  p.tokens = (int)tokens;
  p.n = (int)n;
  p.k = (int)k;
  p.rank = rank;
  p.max_tiles = (int)pl.tiles;
  p.k8 = (int)k8;
  p.rank8 = (rank + 7) & ~7;
  p.splits = pl.splits;
  p.columns = pl.columns;
  p.vector = n % 8 == 0 && base_stride % 8 == 0 && out_stride % 8 == 0 && aligned(base, 16) && aligned(out, 16);
  hipStream_t s = as_stream(stream);
  return dtype == LR_DTYPE_BF16 ? add_by_rank<__bf16>(p, pl, s) : add_by_rank<_Float16>(p, pl, s);
}
