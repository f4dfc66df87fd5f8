// adapters.hip - low-rank adapters of many requests beside a shared projection:
//
//   out[t] = base[t] + scale[a] (x[t] down[a]^T) up[a]^T,   a = index[t], or base[t] without one
//
// with down[a] [rank, k] and up[a] [n, rank]. A plan, made once for a batch and used by
// every layer, lists the tokens by adapter in tiles of at most 64, and the tiles in pairs. Two kernels:
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
constexpr int kFewTokens = 256;     // up to which expand_few runs
// An offset past every buffer here: such a lane reads zeros.
constexpr uint32_t kOutside = 0xfff80000u;
constexpr int64_t kMaxWindow = 0xfff00000ll;

// Tiles that a plan may have: full ones, and one more for each adapter in use.
int64_t plan_tiles(int64_t tokens, int64_t adapters) {
  return tokens / kTokens + (adapters + 1 < tokens ? adapters + 1 : tokens);
}

// Rows of x that the DMAs cannot fetch (of any 2-byte alignment, or that end inside 16 bytes), with
// zeros behind them. A thread per 16 bytes of the copy.
__global__ __launch_bounds__(256) void copy_rows(const uint16_t* x, int64_t stride, int64_t tokens, int k, int k8, uint16_t* to) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int chunks = k8 / 8;
  const int64_t row = i / chunks;
  if (row >= tokens) return;
  const int c = (int)(i - row * chunks) * 8;
  const uint16_t* const from = x + row * stride + c;
  uint4 v;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const uint32_t low = c + e < k ? from[e] : 0, high = c + e + 1 < k ? from[e + 1] : 0;
    set_word(v, e / 2, low | high << 16);
  }
  *reinterpret_cast<uint4*>(to + row * k8 + c) = v;
}

// Whether rows of x, `stride` elements apart, have to be copied.
bool copied(const void* x, int64_t stride, int64_t k) {
  return k % 8 || stride % 8 || !aligned(x, 16) || stride >= (1LL << 30) || (stride > 0 && stride < k);
}

// -------------------------------------------------------------------- plan ----
constexpr int kPlan = 1024;   // threads

// A counting sort by one workgroup: every wave counts its stretch of the tokens, then puts
// them in their places in order. Tokens without an adapter (an index outside 0 .. adapters - 1)
// come last, as those of adapter -1. Latency bounds it, once per batch: 4 us for one token, 25 for 12605.
__global__ __launch_bounds__(kPlan) void plan_adapters(const int32_t* index, int tokens, int adapters, int32_t* order,
                                                       int4* tiles, int max_tiles) {
  constexpr int WAVES = kPlan / 64;
  extern __shared__ int counts[];   // [WAVES][adapters + 1]: tokens, then their next place
  __shared__ int sums[3][WAVES];
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
  // Thread t has kinds 2 t and 2 t + 1: their tokens, tiles and pairs of tiles, and those before them.
  int n[2] = {0, 0}, need[2], pairs[2];
  for (int j = 0; j < 2; ++j) {
    const int a = 2 * t + j;
    if (a < kinds)
      for (int w = 0; w < WAVES; ++w) n[j] += counts[w * kinds + a];
    need[j] = (n[j] + kTokens - 1) / kTokens;
    pairs[j] = a < adapters ? (need[j] + 1) / 2 : 0;
  }
  const int upto_n = wave_prefix_sum(n[0] + n[1]), upto_t = wave_prefix_sum(need[0] + need[1]);
  const int upto_p = wave_prefix_sum(pairs[0] + pairs[1]);
  if (lane == 63) {
    sums[0][wave] = upto_n;
    sums[1][wave] = upto_t;
    sums[2][wave] = upto_p;
  }
  __syncthreads();
  int place = upto_n - n[0] - n[1], tile = upto_t - need[0] - need[1], all = 0;
  int pair = upto_p - pairs[0] - pairs[1], all_pairs = 0;
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) {
      place += sums[0][w];
      tile += sums[1][w];
      pair += sums[2][w];
    }
    all += sums[1][w];
    all_pairs += sums[2][w];
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
    for (int i = 0; i < need[j]; ++i) {
      int4& to = tiles[tile + i];
      to.x = a < adapters ? a : -1;
      to.y = place + i * kTokens;
      to.z = min(kTokens, n[j] - i * kTokens);
    }
    for (int i = 0; i < pairs[j]; ++i) tiles[pair + i].w = tile + 2 * i;
    pair += pairs[j];
    place += n[j];
    tile += need[j];
  }
  for (int i = all + t; i < max_tiles; i += kPlan) {
    tiles[i].x = -1;
    tiles[i].y = tiles[i].z = 0;
  }
  for (int i = all_pairs + t; i < max_tiles; i += kPlan) tiles[i].w = -1;
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
  int tokens, n, k, rank, max_tiles, max_pairs;
  int k8, rank8;         // rows of down and up, in elements
  int splits;            // of k
  int columns;           // of a workgroup of expand
};

__device__ __forceinline__ void dma16s(__amdgpu_buffer_rsrc_t rsrc, void* lds, uint32_t voffset, uint32_t soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)lds, 16, voffset, soffset, 0, 0);
}

// Workgroups are dealt to the 8 XCDs in turn; here each XCD takes a contiguous run of tiles, so
// that its L2 serves an adapter to the tiles that share it (3683 tokens, 5376 columns, rank 64:
// 14.6 us without, 13.2 so).
__device__ __forceinline__ uint32_t run_of_xcd() {
  const uint32_t per = gridDim.x >> 3, rest = gridDim.x & 7, xcd = blockIdx.x & 7;
  return (xcd < rest ? xcd * (per + 1) : rest * (per + 1) + (xcd - rest) * per) + (blockIdx.x >> 3);
}

template <int COUNT>
__device__ __forceinline__ void wait_loads() {   // all but the last COUNT
  static_assert(COUNT < 64, "vmcnt");
  __builtin_amdgcn_s_waitcnt((COUNT & 15) | (COUNT >> 4) << 14 | 0x70 | 0xf00);
}

// Slots of the rings: three, two and one workgroups per CU.
template <int RP, bool PAIR>
constexpr int kRingX = RP == 32 ? 5 : (RP == 64 ? 6 : (PAIR ? 4 : 8));
template <int RP>
constexpr int kRingD = RP == 32 ? 3 : 4;

// Four waves; steps of 64 columns through rings of LDS slots that hold 64 rows of x or RP of
// down, 128 bytes each (16-byte chunk c of row r in place c ^ r / 2 % 8). Wave w takes the columns
// 16 w .. of a step for all rows, so that each element leaves the LDS once; the waves' sums are
// added at the end. The product is transposed, down x^T: a lane holds four ranks of a token
// next to each other.
// (One array holds all of a kernel's LDS: between two the compiler cannot tell which a DMA
// writes, and waits for all of them before any read. With a second one 12605 x 14336 at
// rank 128 took 285 us.)
// What it takes in stays at 32 to 40 KB/us per CU whatever the rings' depth, and at rank 128 down is
// two thirds of it. PAIR: two tiles of an adapter at a time, so that down comes half as often (12605
// tokens of four adapters, 14336 columns at rank 128, with an expand of 128 columns: 117 us, 138
// a tile at a time).
template <typename T, int RP, bool PAIR>
__global__ __launch_bounds__(256) void shrink(AdapterArgs p) {
  typedef typename Mfma<T>::V V8;
  constexpr int TOKENS = PAIR ? 2 * kTokens : kTokens;
  constexpr int RB = RP / 32, TB = TOKENS / 32, ROW = 2 * kStep, RX = kRingX<RP, PAIR>, RD = kRingD<RP>, CH = ROW / 16, PER = 1024 / ROW;
  constexpr int SX = TOKENS * ROW, SD = RP * ROW, LDS = RX * SX + RD * SD, XD = TOKENS / PER / 4, DD = RP / PER / 4;   // DMAs of a wave
  constexpr int GROUP = 4 < TB * RB ? 4 : TB * RB;   // blocks that are added at a time
  static_assert(LDS >= 4 * GROUP * 4096, "the sums take the rings' place");
  __shared__ __attribute__((aligned(1024))) char smem[LDS];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int half = lane >> 5, col = lane & 31;
  const uint32_t id = run_of_xcd(), places = (uint32_t)(PAIR ? p.max_pairs : p.max_tiles);
  const int place = (int)(id % places), split = (int)(id / places), tile = PAIR ? p.tiles[place].w : place;
  if (PAIR && tile < 0) return;
  const int4 info = p.tiles[tile];
  const int a = info.x, start = info.y;
  int count = info.z;
  if (a < 0 || count == 0) return;
  if (PAIR && tile + 1 < p.max_tiles) {
    // (The first of two is full, so that their tokens, and their rows of inner, are in line.)
    const int4 next = p.tiles[tile + 1];
    count += next.x == a ? next.z : 0;
  }
  const int steps = (p.k + kStep - 1) / kStep, chunk = (steps + p.splits - 1) / p.splits;
  const int s0 = min(steps, split * chunk), s1 = min(steps, s0 + chunk);
  const __amdgpu_buffer_rsrc_t xr = row_rsrc(p.x + p.first * p.xs, ((int64_t)(p.window - 1) * p.xs + p.k8) * 2);
  const __amdgpu_buffer_rsrc_t dr = row_rsrc(p.down + (int64_t)a * p.rank * p.k8, (int64_t)p.rank * p.k8 * 2);
  // This lane's rows and chunk of each DMA: chunk c of row r lies in place c ^ turn(r).
  uint32_t xo[XD], dof[DD];
  auto turn = [](int r) __attribute__((always_inline)) { return r * ROW / 256 % CH; };
#pragma unroll
  for (int i = 0; i < XD; ++i) {
    const int r = (wave * XD + i) * PER + lane / CH;
    const int64_t tok = r < count ? p.order[start + r] - p.first : -1;
    const bool in = tok >= 0 && tok < p.window;
    xo[i] = in ? (uint32_t)(tok * p.xs * 2) : kOutside;
  }
#pragma unroll
  for (int i = 0; i < DD; ++i) {
    const int r = (wave * DD + i) * PER + lane / CH;
    dof[i] = r < p.rank ? (uint32_t)((int64_t)r * p.k8 * 2) : kOutside;
  }
  // Steps of whole chunks take a scalar offset; in others those past the last column, or all of
  // them past the last step, read as zero on both sides.
  const int full = min(s1, p.k8 / kStep);
  auto load = [&](__amdgpu_buffer_rsrc_t from, char* lds, uint32_t row, int r, int s) __attribute__((always_inline)) {
    const int c = (lane % CH ^ turn(r)) * 8;
    if (s < full) dma16s(from, lds, row == kOutside ? kOutside : row + c * 2, (uint32_t)s * (kStep * 2));
    else dma16(from, lds, s < s1 && s * kStep + c < p.k8 && row != kOutside ? row + (s * kStep + c) * 2 : kOutside);
  };
  int slot_x = 0, slot_d = 0;   // that the next step goes to
  auto issue_x = [&](int s) {
#pragma unroll
    for (int i = 0; i < XD; ++i) load(xr, smem + slot_x * SX + (wave * XD + i) * 1024, xo[i], (wave * XD + i) * PER + lane / CH, s);
    slot_x = slot_x + 1 == RX ? 0 : slot_x + 1;
  };
  auto issue_d = [&](int s) {
#pragma unroll
    for (int i = 0; i < DD; ++i)
      load(dr, smem + RX * SX + slot_d * SD + (wave * DD + i) * 1024, dof[i], (wave * DD + i) * PER + lane / CH, s);
    slot_d = slot_d + 1 == RD ? 0 : slot_d + 1;
  };
  v16f acc[TB][RB];
#pragma unroll
  for (int b = 0; b < TB; ++b)
#pragma unroll
    for (int c = 0; c < RB; ++c)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[b][c][e] = 0.0f;
  // Step s issues x(s + RX - 1) and then down(s + RD - 1); before the first one:
#pragma unroll
  for (int i = 0; i < RX - RD; ++i) issue_x(s0 + i);
#pragma unroll
  for (int i = 0; i < RD - 1; ++i) {
    issue_x(s0 + RX - RD + i);
    issue_d(s0 + i);
  }
  // A step's fragments are read while the one before is multiplied.
  auto steps_of = [&](auto blocks) {   // of 32 tokens
    constexpr int B = decltype(blocks)::value, PARTS = kStep / 64;
    V8 df[2][PARTS][RB], xf[2][PARTS][B];
    int read_x = 0, read_d = 0;
    auto fetch = [&](V8 (&d)[PARTS][RB], V8 (&x)[PARTS][B]) __attribute__((always_inline)) {
      const char* const xs = smem + read_x * SX;
      const char* const ds = smem + RX * SX + read_d * SD;
#pragma unroll
      for (int i = 0; i < PARTS; ++i) {
        // (All rows of a block have the turn of the first: 32 rows are whole turns.)
        const int place = ((8 * i + 2 * wave + half) ^ turn(col)) * 16;
#pragma unroll
        for (int c = 0; c < RB; ++c) d[i][c] = *reinterpret_cast<const V8*>(ds + (32 * c + col) * ROW + place);
#pragma unroll
        for (int b = 0; b < B; ++b) x[i][b] = *reinterpret_cast<const V8*>(xs + (32 * b + col) * ROW + place);
      }
      read_x = read_x + 1 == RX ? 0 : read_x + 1;
      read_d = read_d + 1 == RD ? 0 : read_d + 1;
    };
    auto arrive = [&](auto left) __attribute__((always_inline)) {
      wait_loads<decltype(left)::value>();
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    auto step = [&](V8 (&d)[PARTS][RB], V8 (&x)[PARTS][B], V8 (&nd)[PARTS][RB], V8 (&nx)[PARTS][B], int s)
        __attribute__((always_inline)) {
      // Step s + 1 is there, and every wave is done with step s - 1, whose slots are next.
      arrive(std::integral_constant<int, (RD - 3) * (XD + DD)>{});
      issue_x(s + RX - 1);
      issue_d(s + RD - 1);
      fetch(nd, nx);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < PARTS; ++i)
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
          for (int c = 0; c < RB; ++c) acc[b][c] = Mfma<T>::mul(d[i][c], x[i][b], acc[b][c]);
      __builtin_amdgcn_sched_barrier(0);
    };
    arrive(std::integral_constant<int, (RD - 2) * (XD + DD)>{});
    fetch(df[0], xf[0]);
    int s = s0;
#pragma unroll 1
    for (; s + 1 < s1; s += 2) {
      step(df[0], xf[0], df[1], xf[1], s);
      step(df[1], xf[1], df[0], xf[0], s + 1);
    }
    if (s < s1) step(df[0], xf[0], df[1], xf[1], s);
  };
  if (!PAIR && count <= TOKENS / 2) steps_of(std::integral_constant<int, TB / 2>{});
  else steps_of(std::integral_constant<int, TB>{});
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
        const int64_t of = p.order[start + tok] - p.first;
        if (of < 0 || of >= p.window) continue;
      }
      *reinterpret_cast<float4*>(part + tok * RP + r) = v;
    }
  }
}

// ------------------------------------------------------------------ expand ----
// inner: the shares of k added up in order, in place of the first one. A thread per four ranks
// (3683 tokens at rank 64: 4.6 us, most of it the launch and one way to memory and back).
template <int RP>
__global__ __launch_bounds__(256) void add_shares(AdapterArgs p) {
  const int at = (int)(blockIdx.x * 256 + threadIdx.x), tile = at / (kTokens * RP / 4), tok = at / (RP / 4) % kTokens;
  if (tile >= p.max_tiles || p.tiles[tile].x < 0 || tok >= p.tiles[tile].z) return;
  float4* const to = reinterpret_cast<float4*>(p.part) + at;
  const int64_t share = (int64_t)p.max_tiles * kTokens * RP / 4;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  constexpr int COUNT = 8;   // on their way at a time
  for (int s = 0; s < p.splits; s += COUNT) {
    float4 y[COUNT];
#pragma unroll
    for (int i = 0; i < COUNT; ++i) y[i] = s + i < p.splits ? to[(s + i) * share] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      v.x += y[i].x;
      v.y += y[i].y;
      v.z += y[i].z;
      v.w += y[i].w;
    }
  }
  *to = v;
}

// The power of two that takes a row's largest to [1, 2); 0 for one that is zero or infinite.
__device__ __forceinline__ int exponent_of(float top) {
  return top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 1 : 0;
}

// v * 2^-ex as numbers of the type and what their rounding leaves. An infinity has no rest.
template <typename T>
__device__ __forceinline__ void split8(const float* v, int ex, uint4& hi, uint4& lo) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float y0 = __builtin_amdgcn_ldexpf(v[2 * j], -ex), y1 = __builtin_amdgcn_ldexpf(v[2 * j + 1], -ex);
    const uint32_t w = Mfma<T>::pack(y0, y1);
    const float d0 = y0 - Mfma<T>::first(w), d1 = y1 - Mfma<T>::second(w);
    set_word(hi, j, w);
    set_word(lo, j, Mfma<T>::pack(__builtin_fabsf(y0) < INFINITY ? d0 : 0.0f, __builtin_fabsf(y1) < INFINITY ? d1 : 0.0f));
  }
}

// Few tokens, most tiles with one or some: what counts is the stream of up's rows. Every wave has
// its quarter of the columns, 32 at a time, straight in registers; a lane adds four columns of its
// token at a time. The waves add up inner's shares together, a quarter of them each. Tiles of
// more than 32 tokens take two turns. (All of a workgroup's rows sent to LDS at once instead: 22.7
// against 20.4 us with shrink, 64 tokens of 32 adapters, 5120 to 15360 columns at rank 32.)
template <typename T, int RP, bool VECTOR>
__global__ __launch_bounds__(256, VECTOR && RP < 128 ? (RP == 32 ? 3 : 2) : 1) void expand_few(AdapterArgs p) {
  typedef typename Mfma<T>::V V8;
  constexpr int KR = RP / 16, BLOCKS = 2;   // of 32 columns on their way
  __shared__ float4 sums[4][32][RP / 4 + 1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int half = lane >> 5, col = lane & 31;
  const int tile = (int)(blockIdx.x % (uint32_t)p.max_tiles), run = (int)(blockIdx.x / (uint32_t)p.max_tiles);
  const int4 info = p.tiles[tile];
  const int a = info.x, count = info.z, quarter = p.columns / 4;
  const int first = run * p.columns + wave * quarter, last = min(p.n, first + quarter);
  if (count == 0 || (a < 0 && p.out == p.base)) return;
  const uint16_t* const up = p.up + (int64_t)(a < 0 ? 0 : a) * p.n * p.rank8;
  const float scale = p.scale[a < 0 ? 0 : a];
  for (int t0 = 0; t0 < count; t0 += 32) {
    const bool mine = t0 + col < count;
    const int row = min(t0 + col, count - 1);
    const int64_t tok = p.order[info.y + row];
    const uint16_t* const base = p.base + tok * p.bs;
    uint16_t* const out = p.out + tok * p.os;
    V8 uf[BLOCKS][KR];
    auto load = [&](int n) {
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const uint16_t* const from = up + (int64_t)min(n + 32 * b + col, p.n - 1) * p.rank8;
#pragma unroll
        for (int d = 0; d < KR; ++d) {
          const int r = 16 * d + 8 * half;
          uf[b][d] = *reinterpret_cast<const V8*>(from + (r < p.rank8 ? r : 0));   // (inner is 0 there)
        }
      }
    };
    // The lane's token, ranks 16 d + 8 half + 0 .. 7.
    V8 hi[KR], lo[KR];
    float back = 1.0f;
    if (a >= 0) {
      load(min(first, p.n - 1));
      float v[KR][8], top = 0.0f;
      const float* const from = p.part + ((int64_t)tile * kTokens + row) * RP + 8 * half;
      const int64_t share = (int64_t)p.max_tiles * kTokens * RP;
#pragma unroll
      for (int d = 0; d < KR; ++d)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[d][e] = 0.0f;
      for (int s = wave; s < p.splits; s += 4)
#pragma unroll
        for (int d = 0; d < KR; ++d)
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            const float4 y = *reinterpret_cast<const float4*>(from + s * share + 16 * d + e);
            v[d][e] += y.x;
            v[d][e + 1] += y.y;
            v[d][e + 2] += y.z;
            v[d][e + 3] += y.w;
          }
      if (t0) __syncthreads();   // the tokens before have been read
#pragma unroll
      for (int d = 0; d < KR; ++d)
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          sums[wave][col][4 * d + 2 * half + e / 4] = make_float4(v[d][e], v[d][e + 1], v[d][e + 2], v[d][e + 3]);
      __syncthreads();
#pragma unroll
      for (int d = 0; d < KR; ++d)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          float4 y = sums[0][col][4 * d + 2 * half + e / 4];
#pragma unroll
          for (int w = 1; w < 4; ++w) {
            const float4 z = sums[w][col][4 * d + 2 * half + e / 4];
            y.x += z.x;
            y.y += z.y;
            y.z += z.z;
            y.w += z.w;
          }
          *reinterpret_cast<float4*>(&v[d][e]) = y;
        }
#pragma unroll
      for (int d = 0; d < KR; ++d)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[d][e] = 16 * d + 8 * half + e < p.rank ? v[d][e] * scale : 0.0f;   // (a row past the rank may hold 0 * infinity)
          top = fmaxf(top, __builtin_fabsf(v[d][e]));
        }
      const int ex = exponent_of(max_with_partner(top));
      back = __builtin_amdgcn_ldexpf(1.0f, ex);
#pragma unroll
      for (int d = 0; d < KR; ++d) {
        uint4 h, l;
        split8<T>(v[d], ex, h, l);
        hi[d] = __builtin_bit_cast(V8, h);
        lo[d] = __builtin_bit_cast(V8, l);
      }
    }
    for (int n = first; n < last; n += 32 * BLOCKS) {
      uint2 kept[BLOCKS][4];
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int at = n + 32 * b + 8 * g + 4 * half;
          if constexpr (VECTOR) {
            kept[b][g] = *reinterpret_cast<const uint2*>(base + min(at, last - 4));
          } else {
            kept[b][g].x = base[min(at, last - 1)] | (uint32_t)base[min(at + 1, last - 1)] << 16;
            kept[b][g].y = base[min(at + 2, last - 1)] | (uint32_t)base[min(at + 3, last - 1)] << 16;
          }
        }
      v16f s[BLOCKS];
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[b][e] = 0.0f;
        if (a < 0) continue;
#pragma unroll
        for (int d = 0; d < KR; ++d) {
          s[b] = Mfma<T>::mul(uf[b][d], lo[d], s[b]);
          s[b] = Mfma<T>::mul(uf[b][d], hi[d], s[b]);
        }
      }
      if (a >= 0 && n + 32 * BLOCKS < last) load(n + 32 * BLOCKS);
      if (!mine) continue;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int at = n + 32 * b + 8 * g + 4 * half;
          if (at >= last) continue;
          uint2 w = kept[b][g];
          if (a >= 0) {
            w.x = Mfma<T>::pack(Mfma<T>::first(w.x) + s[b][4 * g] * back, Mfma<T>::second(w.x) + s[b][4 * g + 1] * back);
            w.y = Mfma<T>::pack(Mfma<T>::first(w.y) + s[b][4 * g + 2] * back, Mfma<T>::second(w.y) + s[b][4 * g + 3] * back);
          }
          if constexpr (VECTOR) {
            *reinterpret_cast<uint2*>(out + at) = w;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (at + e < last) out[at + e] = (uint16_t)((e < 2 ? w.x : w.y) >> (16 * (e & 1)));
          }
        }
    }
  }
}

// Four waves: 32 tokens x 64 columns each of a step of 128 columns. up's rows come through
// LDS like the keys of lr_attention.h (a row holds RP numbers); the sums leave through LDS
// too, so that base and out are read and written in whole lines. VECTOR: 16 bytes at a time.
// (3683 tokens, 28672 columns at rank 64: 93-97 us, 4.6 TB/s.)
template <typename T, int RP, bool VECTOR>
__global__ __launch_bounds__(256) void expand(AdapterArgs p) {
  typedef typename Mfma<T>::V V8;
  constexpr int ROW = 2 * RP, CH = ROW / 16, RPB = 256 / ROW, PAIRS = ROW / 32, KR = RP / 16;
  constexpr int UP = kColumns * ROW, DMAS = UP / 1024 / 4, PITCH = kColumns + 4;
  constexpr int INNER = 2 * kTokens * ROW;   // rounded and rest
  constexpr int OUT = kTokens * PITCH * 4;
  constexpr int RESULT = OUT > INNER ? OUT : INNER;
  __shared__ __attribute__((aligned(1024))) char smem[UP + RESULT + kTokens * 8];
  char* const inner = smem + UP;
  float* const result = reinterpret_cast<float*>(smem + UP);
  float* const exponents = reinterpret_cast<float*>(smem + UP + RESULT);
  int* const tokens = reinterpret_cast<int*>(exponents + kTokens);
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const int half = lane >> 5, col = lane & 31;
  const int tile = (int)(blockIdx.x % (uint32_t)p.max_tiles), run = (int)(blockIdx.x / (uint32_t)p.max_tiles);
  const int4 info = p.tiles[tile];
  const int a = info.x, count = info.z;
  if (count == 0 || (a < 0 && p.out == p.base)) return;
  const int n0 = run * p.columns, n1 = min(p.n, n0 + p.columns);
  if (t < kTokens) tokens[t] = p.order[info.y + min(t, count - 1)];
  // Step c: this thread's row (16 threads of 8 columns each, 16 rows at a time) of base.
  const int c8 = (t & 15) * 8, row0 = t >> 4;
  uint4 kept[kTokens / 16];
  auto load_base = [&](int c) {
#pragma unroll
    for (int i = 0; i < kTokens / 16; ++i) {
      // What lies outside repeats the last row and columns: a load that is left out would
      // cost copies, and with them a wait, where the loop closes.
      const uint16_t* const row = p.base + tokens[16 * i + row0] * p.bs;
      if constexpr (VECTOR) kept[i] = load_nt(reinterpret_cast<const uint4*>(row + min(c + c8, n1 - 8)));
      else
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          set_word(kept[i], e / 2, row[min(c + c8 + e, n1 - 1)] | (uint32_t)row[min(c + c8 + e + 1, n1 - 1)] << 16);
    }
  };
  auto store_out = [&](int c, const uint4 (&from)[kTokens / 16]) {
#pragma unroll
    for (int i = 0; i < kTokens / 16; ++i) {
      const int r = 16 * i + row0, n = c + c8;
      if (r >= count || n >= n1) continue;
      uint16_t* const to = p.out + tokens[r] * p.os + n;
      if constexpr (VECTOR) store_nt(reinterpret_cast<uint4*>(to), from[i]);
      else
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < n1) to[e] = (uint16_t)(word(from[i], e / 2) >> (16 * (e & 1)));
    }
  };
  __syncthreads();
  if (a < 0) {
    for (int c = n0; c < n1; c += kColumns) {
      load_base(c);
      store_out(c, kept);
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
    for (int e = 0; e < EACH; e += 4)
      *reinterpret_cast<float4*>(v + e) =
          tok < count ? *reinterpret_cast<const float4*>(p.part + ((int64_t)tile * kTokens + tok) * RP + r0 + e)
                      : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float scale = p.scale[a];
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      v[e] = r0 + e < p.rank ? v[e] * scale : 0.0f;   // (a row past the rank may hold 0 * infinity)
      top = fmaxf(top, __builtin_fabsf(v[e]));
    }
    top = fmaxf(top, xor_partner<1>(top));
    top = fmaxf(top, xor_partner<2>(top));
    const int ex = exponent_of(top);
    if ((t & 3) == 0) exponents[tok] = __builtin_amdgcn_ldexpf(1.0f, ex);
#pragma unroll
    for (int e = 0; e < EACH; e += 8) {
      uint4 hi, lo;
      split8<T>(v + e, ex, hi, lo);
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
    // Up's rows and base are there; the stores of the step before, which come behind them
    // (four per thread of a full tile), may be on their way.
    if (VECTOR && count == kTokens && c > n0) wait_loads<kTokens / 16>();
    else wait_loads<0>();
    __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): inner, or the step before, has been read
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
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
    __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): the sums are written, up's rows read
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // The sums leave the LDS before the next DMA, for which the compiler would wait otherwise.
    uint4 sum[kTokens / 16];
#pragma unroll
    for (int i = 0; i < kTokens / 16; ++i) {
      const int r = 16 * i + row0;
      const float4 y0 = *reinterpret_cast<const float4*>(result + r * PITCH + c8);
      const float4 y1 = *reinterpret_cast<const float4*>(result + r * PITCH + c8 + 4);
      const float y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t w = word(kept[i], e);
        set_word(sum[i], e, Mfma<T>::pack(Mfma<T>::first(w) + y[2 * e], Mfma<T>::second(w) + y[2 * e + 1]));
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (c + kColumns < n1) {
      issue(c + kColumns);
      load_base(c + kColumns);
    }
    __builtin_amdgcn_sched_barrier(0);
    store_out(c, sum);
    __builtin_amdgcn_sched_barrier(0);
  }
}

struct AddPlan {
  int rank;      // padded
  int splits, columns;
  bool few, pair;
  int64_t tiles, pairs, bytes;
};

AddPlan add_plan(int64_t tokens, int64_t n, int64_t k, int rank, int64_t adapters) {
  AddPlan pl;
  pl.rank = rank <= 32 ? 32 : (rank <= 64 ? 64 : 128);
  pl.tiles = plan_tiles(tokens, adapters);
  const int64_t cus = compute_units(), steps = (k + kStep - 1) / kStep;
  // Columns of an expanding workgroup: up to 1024, less where that leaves fewer than two
  // workgroups per CU; one for few tokens, where each of them adds up the shares (64 tokens of
  // 32 adapters, 15360 columns at rank 32: 19.4 us so, 21.8 with two; 16 tokens 12.0 and 14.3).
  pl.few = tokens <= kFewTokens;
  int64_t c = 1024;
  while (c > kColumns && pl.tiles * ((n + c - 1) / c) < (pl.few ? cus : 2 * cus)) c /= 2;
  pl.columns = (int)c;
  // Shares of k, of four steps and more: what the rounds of workgroups take, their steps at
  // 45 KB/us for each CU and six of them to fill the ring, against a launch to add the shares
  // and their way through memory.
  const int per_cu = pl.rank == 32 ? 3 : (pl.rank == 64 ? 2 : 1);
  // Pairs of tiles where an adapter has seven and more on average, and each CU 30 steps and more.
  // With 640 outputs, a tile at a time and so: 12605 tokens of 4 adapters, 2048 columns (25 steps
  // per CU) 43 and 48 us, 5376 (66) 68 and 65, 7168 (88) 82 and 77, 14336 (176) 142 and 121; 4096 of
  // 4, 5376 (23) level, 7168 (30) 38 and 37, 14336 (60) 53 and 47; 3683 of 8, 7 tiles each, 7168
  // (29) 38 and 37, 20480 (82) 75 and 61; 4096 of 16, 4 tiles each, 10240 (51) 45 and 46, 20480 (101) level.
  pl.pair = pl.rank == 128 && tokens >= 7 * kTokens * adapters && pl.tiles * steps >= 30 * cus;
  pl.pairs = tokens / (2 * kTokens) + (adapters < tokens ? adapters : tokens);
  const int64_t tiles = pl.pair ? pl.pairs : pl.tiles;
  const double step = per_cu * ((pl.pair ? 2 : 1) * kTokens + pl.rank) * 2.0 * kStep / 45e3;
  const double share = (double)pl.tiles * kTokens * pl.rank * 4 * 2.0 / 5e6;
  double least = 0.0;
  for (int s = 1; s <= 16 && (s == 1 || s <= steps / 4); ++s) {
    const double rounds = ceil((double)(tiles * s) / (double)(cus * per_cu));
    const double us = rounds * ((double)((steps + s - 1) / s) + 6.0) * step + (s > 1 ? 2.5 + s * share : 0.0);
    if (s == 1 || us < least) {
      least = us;
      pl.splits = s;
    }
  }
  pl.bytes = pl.splits * pl.tiles * kTokens * pl.rank * 4;
  return pl;
}

template <typename T, int RP>
int add(AdapterArgs p, const AddPlan& pl, bool vector, hipStream_t s) {
  const int64_t rows = kMaxWindow / (p.xs * 2 > 2 * p.k8 ? p.xs * 2 : 2 * p.k8);
  for (int64_t first = 0; first < p.tokens; first += rows) {
    p.first = first;
    p.window = (int)(p.tokens - first < rows ? p.tokens - first : rows);
    if (RP == 128 && pl.pair) shrink<T, RP, RP == 128><<<(unsigned)(pl.pairs * pl.splits), 256, 0, s>>>(p);
    else shrink<T, RP, false><<<(unsigned)(pl.tiles * pl.splits), 256, 0, s>>>(p);
    if (int rc = check_launch("adapter_add")) return rc;
  }
  const unsigned grid = (unsigned)(pl.tiles * ((p.n + pl.columns - 1) / pl.columns));
  if (pl.splits > 1 && !pl.few) {
    add_shares<RP><<<(unsigned)((pl.tiles * (kTokens * RP / 4) + 255) / 256), 256, 0, s>>>(p);
    if (int rc = check_launch("adapter_add")) return rc;
  }
  if (pl.few && vector) expand_few<T, RP, true><<<grid, 256, 0, s>>>(p);
  else if (pl.few) expand_few<T, RP, false><<<grid, 256, 0, s>>>(p);
  else if (vector) expand<T, RP, true><<<grid, 256, 0, s>>>(p);
  else expand<T, RP, false><<<grid, 256, 0, s>>>(p);
  return check_launch("adapter_add");
}

template <typename T>
int add_by_rank(const AdapterArgs& p, const AddPlan& pl, bool vector, hipStream_t s) {
  if (pl.rank == 32) return add<T, 32>(p, pl, vector, s);
  if (pl.rank == 64) return add<T, 64>(p, pl, vector, s);
  return add<T, 128>(p, pl, vector, s);
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

extern "C" int lr_adapter_workspace(int64_t tokens, int64_t n, int64_t k, int rank, int adapters, int copies,
                                    int64_t* bytes) {
  if (int rc = check_add(tokens, n, k, rank, adapters)) return rc;
  LR_REQUIRE(bytes, "adapter_add: null pointer");
  *bytes = tokens ? add_plan(tokens, n, k, rank, adapters).bytes + (copies ? tokens * ((k + 7) & ~7LL) * 2 : 0) : 0;
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
  LR_REQUIRE(aligned(x, 2) && aligned(down, 16) && aligned(up, 16) && aligned(scale, 4) && aligned(order, 4) &&
                 aligned(tiles, 16) && aligned(base, 2) && aligned(out, 2),
             "adapter_add: adapters and plans must be 16-byte aligned");
  const int64_t k8 = (k + 7) & ~7LL;
  LR_REQUIRE(x_stride >= 0 && base_stride >= 0 && (out_stride >= n || tokens == 1),
             "adapter_add: rows of %lld columns %lld apart", (long long)n, (long long)out_stride);
  // What is read by all of the tokens may not change under them.
  auto apart = [&](const void* p, int64_t bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), o = reinterpret_cast<uintptr_t>(out);
    return a + bytes <= o || o + ((tokens - 1) * out_stride + n) * 2 <= a;
  };
  const int64_t rank8 = (rank + 7) & ~7;
  LR_REQUIRE(apart(down, adapters * rank * k8 * 2) && apart(up, adapters * n * rank8 * 2) && apart(scale, adapters * 4) &&
                 apart(order, tokens * 4) && apart(tiles, plan_tiles(tokens, adapters) * 16),
             "adapter_add: out must not overlap the adapters or the plan");
  const bool copies = copied(x, x_stride, k);
  const AddPlan pl = add_plan(tokens, n, k, rank, adapters);
  const int64_t runs = (n + pl.columns - 1) / pl.columns;
  LR_REQUIRE(pl.tiles * pl.splits <= kMaxBlocks && pl.tiles * runs <= kMaxBlocks,
             "adapter_add: %lld tiles of tokens are not supported", (long long)pl.tiles);
  const int64_t needs = pl.bytes + (copies ? tokens * k8 * 2 : 0);
  LR_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= needs,
             "adapter_add: needs a workspace of %lld bytes", (long long)needs);
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
  p.max_pairs = (int)pl.pairs;
  p.k8 = (int)k8;
  p.rank8 = (int)rank8;
  p.splits = pl.splits;
  p.columns = pl.columns;
  const bool vector = n % 8 == 0 && base_stride % 8 == 0 && out_stride % 8 == 0 && aligned(base, 16) && aligned(out, 16);
  hipStream_t s = as_stream(stream);
  if (copies) {
    const int64_t blocks = (tokens * (k8 / 8) + 255) / 256;
    LR_REQUIRE(blocks <= kMaxBlocks, "adapter_add: %lld x %lld inputs to copy are not supported", (long long)tokens, (long long)k);
    uint16_t* const to = reinterpret_cast<uint16_t*>(static_cast<char*>(workspace) + pl.bytes);
    copy_rows<<<(unsigned)blocks, 256, 0, s>>>(p.x, p.xs, tokens, p.k, p.k8, to);
    if (int rc = check_launch("adapter_add")) return rc;
    p.x = to;
    p.xs = k8;
  }
  return dtype == LR_DTYPE_BF16 ? add_by_rank<__bf16>(p, pl, vector, s) : add_by_rank<_Float16>(p, pl, vector, s);
}
