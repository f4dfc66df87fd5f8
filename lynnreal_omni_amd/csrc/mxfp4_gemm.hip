// mxfp4_gemm.hip - products of MXFP4 rows on CDNA4's scaled MFMA.
//
//   y[m, n] = sum_b 2^(ea[m, b] + eb[n, b] - 254) sum_{k in block b} A[m, k] W[n, k]
//   out     = bf16(y + bias[n]), or GELU-tanh / gated residual of that bf16 value
//
// A and W are E2M1 codes, ea and eb the E8M0 bytes of their blocks of 32
// (mxfp4.hip). The products of two codes and their scales are exact in fp32;
// v_mfma_scale_f32_16x16x128_f8f6f4 adds them in fp32. y is rounded to bf16
// before the epilogue, so that a fused epilogue gives the bits of the product
// followed by gelu_tanh or _gated_residual, as for the INT8 product.
//
// A lane of the 16x16x128 FP4 MFMA holds 16 bytes of a row, 4 lanes a row's 64
// bytes: byte for byte the operand layout of the 16x16x64 INT8 MFMA, at the same
// cycles and twice the products. So the tile kernels move operands like the INT8
// ones: k-steps of 128 bytes (256 columns) by DMA into XOR-swizzled LDS, read
// back by ds_read_b128. Scales (1/16 of the operands' bytes) go from global
// memory to registers in the order of lr_mxfp4.h, one 8-byte load per 64 rows
// and k-step, a k-step ahead.
#include <type_traits>
#include <utility>

#include "lr_device.h"
#include "lr_mxfp4.h"
#include "lr_mxfp4_rows.h"
#include "lr_runtime.h"

namespace lr {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

struct Fp4Args {
  const uint8_t* a;       // codes [m, kb]
  const uint8_t* as;      // scale tiles
  const uint8_t* b;       // codes [n, kb]
  const uint8_t* bs;
  const uint16_t* bias;   // or null
  uint16_t* c;
  const uint16_t* resid;
  const uint16_t* table;
  const int64_t* indices;
  int64_t m, n, kb;       // kb: bytes of codes per row (a multiple of 16)
  int64_t table_rows, table_width, sequence;
  int gate_slot;
  int col_tiles;          // scale tiles along a row = k-steps
  int tiles_m, tiles_n;
  int staged;             // N % 8 == 0 and 16-byte aligned output (residual, table) rows
};

enum { EPI_BF16 = LR_EPI_BF16, EPI_GELU = LR_EPI_GELU_TANH, EPI_GATED = LR_EPI_GATED_RESIDUAL };

// One scaled MFMA; bytes WO of ws and AO of as hold the lane's scales.
template <int WO, int AO>
__device__ __forceinline__ v4f mfma_fp4(const v4i& w, const v4i& a, const v4f& c, int ws, int as) {
  const v8i w8 = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, a8, c, 4, 4, WO, ws, AO, as);
}

// f(integral_constant<int, 0>), .., f(integral_constant<int, N - 1>): loops whose
// index is an instruction's field.
template <class F, int... I>
__device__ __forceinline__ void each(std::integer_sequence<int, I...>, F f) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F f) {
  each(std::make_integer_sequence<int, N>(), f);
}

// ------------------------------------------------------------ epilogue ----
__device__ __forceinline__ int64_t table_row(const Fp4Args& p, int64_t row) {
  return clamp_index(p.indices[p.sequence >= p.m ? row : row % p.sequence], p.table_rows);
}

// From the bf16 value y to the output.
template <int EPI>
__device__ __forceinline__ float finish(float y, float gate, float x) {
  if (EPI == EPI_GELU) return fast_gelu_tanh(y);
  if (EPI == EPI_GATED) return x + round_bf(gate * y);
  return y;
}

template <int EPI>
__device__ __forceinline__ void store_scalar(const Fp4Args& p, int64_t row, int64_t col, float v) {
  const int64_t o = row * p.n + col;
  if (p.bias) v = v + bf_to_f(p.bias[col]);
  float gate = 0.0f, x = 0.0f;
  if (EPI == EPI_GATED) {
    gate = bf_to_f(p.table[table_row(p, row) * p.table_width + (int64_t)p.gate_slot * p.n + col]);
    x = bf_to_f(p.resid[o]);
  }
  p.c[o] = (uint16_t)(pack_bf2(finish<EPI>(round_bf(v), gate, x), 0.0f) & 0xffffu);
}

template <int EPI>
__device__ __forceinline__ uint4 finish8(const uint4& y, const uint4& gate, const uint4& x) {
  uint4 o;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t u = word(y, w), g = word(gate, w), r = word(x, w);
    set_word(o, w, EPI == EPI_BF16 ? u : pack_bf2(finish<EPI>(bf_lo(u), bf_lo(g), bf_lo(r)),
                                                  finish<EPI>(bf_hi(u), bf_hi(g), bf_hi(r))));
  }
  return o;
}

// A wave's (16 * FM) x (16 * FN) outputs, in the MFMA layout: lane l has row
// 16 * i + l % 16 and columns 16 * j + 4 * (l / 16) + 0..3 of tile (i, j).
// Staged through LDS as bf16 (row pitch 2 * WN + 16 bytes), then row by row, 16
// bytes per lane, so that every store fills whole 128-byte lines (for WN >= 64)
// and the residual and gate rows are read as such.
template <int FM, int FN, int EPI>
__device__ __forceinline__ void store_staged(const Fp4Args& p, const v4f (&acc)[FM][FN], char* stage, int64_t m0,
                                             int64_t n0, int lane) {
  constexpr int WM = 16 * FM, WN = 16 * FN, PITCH = 2 * WN + 16;
  const int lr_ = lane & 15, lg = lane >> 4;
  uint2 bv[FN];
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    const int64_t col = n0 + 16 * j + 4 * lg;
    bv[j] = p.bias ? *reinterpret_cast<const uint2*>(p.bias + (col < p.n ? col : p.n - 4)) : make_uint2(0u, 0u);
  }
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i)
      *reinterpret_cast<uint2*>(stage + (16 * i + lr_) * PITCH + (16 * j + 4 * lg) * 2) =
          make_uint2(pack_bf2(acc[i][j][0] + bf_lo(bv[j].x), acc[i][j][1] + bf_hi(bv[j].x)),
                     pack_bf2(acc[i][j][2] + bf_lo(bv[j].y), acc[i][j][3] + bf_hi(bv[j].y)));
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's staging writes are done
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  constexpr int CPR = WN / 8;                  // 16-byte chunks per row
  constexpr int ITERS = (WM * CPR + 63) / 64;
  // Gated: residual and gate chunks of a batch of rows are loaded together, from
  // clamped addresses, so that no load sits under a branch.
  constexpr int BATCH = ITERS % 4 == 0 ? 4 : (ITERS % 2 == 0 ? 2 : 1);
#pragma unroll 1
  for (int s0 = 0; s0 < ITERS; s0 += BATCH) {
    uint4 v[BATCH], x[BATCH], g[BATCH];
    int64_t o[BATCH];
    bool ok[BATCH];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int q = (s0 + b) * 64 + lane;
      const int r = q / CPR, ch = q % CPR;
      const int64_t row = m0 + r, col = n0 + ch * 8;
      ok[b] = q < WM * CPR && row < p.m && col < p.n;
      o[b] = row * p.n + col;
      v[b] = *reinterpret_cast<const uint4*>(stage + (q < WM * CPR ? r * PITCH + ch * 16 : 0));
      x[b] = g[b] = make_uint4(0u, 0u, 0u, 0u);
      if (EPI == EPI_GATED) {
        const int64_t row_l = ok[b] ? row : (m0 < p.m ? m0 : 0), col_l = ok[b] ? col : 0;
        x[b] = load_nt(reinterpret_cast<const uint4*>(p.resid + row_l * p.n + col_l));
        g[b] = *reinterpret_cast<const uint4*>(p.table + table_row(p, row_l) * p.table_width +
                                               (int64_t)p.gate_slot * p.n + col_l);
      }
    }
#pragma unroll
    for (int b = 0; b < BATCH; ++b)
      if (ok[b]) store_nt(reinterpret_cast<uint4*>(p.c + o[b]), finish8<EPI>(v[b], g[b], x[b]));
  }
}

template <int FM, int FN, int EPI>
__device__ __forceinline__ void store_direct(const Fp4Args& p, const v4f (&acc)[FM][FN], int64_t m0, int64_t n0,
                                             int lane) {
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t row = m0 + 16 * i + (lane & 15), col = n0 + 16 * j + 4 * (lane >> 4) + e;
        if (row < p.m && col < p.n) store_scalar<EPI>(p, row, col, acc[i][j][e]);
      }
}

// ----------------------------------------------------------- tile order ----
// Workgroups are dealt to the 8 XCDs round-robin; each XCD walks a contiguous,
// M-grouped range of tiles so that its L2 holds the panels its CUs share. Groups of
// 2 / 4 / 6 / 8 tiles: 640 / 629 / 630 / 697 us at 16384 x 16384 x 5120, 899 /
// 886 / 888 / 917 at 12605 x 28672 x 5376, within 1% at a single round of tiles.
constexpr int kGroup = 4;
__device__ __forceinline__ void tile_coords(const Fp4Args& p, int pid, int& tm, int& tn) {
  const int total = p.tiles_m * p.tiles_n;
  const int xcd = pid & 7, local = pid >> 3;
  const int q = total >> 3, r = total & 7;
  const int lid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + local;
  const int span = kGroup * p.tiles_n;
  const int g = lid / span;
  const int first = g * kGroup;
  const int gm = min(p.tiles_m - first, kGroup);
  const int within = lid - g * span;
  tm = first + within % gm;
  tn = within / gm;
}

// The vmcnt field of s_waitcnt.
constexpr int vm(int n) { return (n & 15) | (n >> 4) << 14; }

typedef __attribute__((address_space(3))) void* lds_ptr_t;
// 16 bytes per lane from a buffer straight into LDS at lds + 16 * lane; offsets
// past the buffer's end read as zero.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rsrc, void* lds, uint32_t voffset, uint32_t soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)lds, 16, voffset, soffset, 0, 0);
}

// The same with 4 bytes per lane.
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t rsrc, void* lds, uint32_t voffset, uint32_t soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)lds, 4, voffset, soffset, 0, 0);
}

// The scale registers of 16 * F rows for one k-step: eight bytes per 64 rows. Rows
// that do not start at a multiple of 64 (START: what their first is a multiple of)
// take one more load, and settle() moves their bytes down. Byte byte(f, h) of
// w[f / 2] is then fragment f, half h.
template <int F, int START>
struct Scales {
  static constexpr int kLoads = F == 2 ? 1 : (F * 16 + 64 - START + 63) / 64, kWords = F == 2 ? 1 : 2 * kLoads;
  static constexpr int byte(int f, int h) { return 2 * (f & 1) + h; }
  static_assert(START == 16 || START == 32 || START == 64, "first row");
  uint32_t w[kWords];
  // rsrc: the panel's scale tiles; groups: how many of 64 rows it has; row: of the
  // first of the rows in it. Rows past the panel (past the operand's last, whose
  // codes read as zero) repeat its last group. All but the lane's offset is scalar.
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rsrc, int groups, int row, int col_tiles, int kt,
                                       int lane) {
#pragma unroll
    for (int t = 0; t < kLoads; ++t) {
      const int at = (min((row >> 6) + t, groups - 1) * col_tiles + kt) * 512;
      if (F == 2) {
        w[0] = __builtin_amdgcn_raw_buffer_load_b32(rsrc, lane * 8, at + ((row >> 4) & 2) * 2, 0);
      } else {
        const v2u v = __builtin_amdgcn_raw_buffer_load_b64(rsrc, lane * 8, at, 0);
        w[2 * t] = v.x;
        w[2 * t + 1] = v.y;
      }
    }
  }
  __device__ __forceinline__ void settle(int row) {
    if (F == 2 || START == 64) return;
    // Here and not behind the load, where it would wait for it.
#pragma unroll
    for (int i = 0; i < kWords; ++i) asm volatile("" : "+v"(w[i]));
    const uint32_t words = row & 32 ? 0xffffffffu : 0u;
    const int bits = START == 16 ? row & 16 : 0;
#pragma unroll
    for (int i = 0; i < kWords - 1; ++i) w[i] ^= (w[i] ^ w[i + 1]) & words;
    if (START == 16) {
#pragma unroll
      for (int i = 0; i < kWords - 1; ++i) w[i] = __builtin_amdgcn_alignbit(w[i + 1], w[i], bits);
    }
  }
};

// ---------------------------------------------------------- tile kernel ----
// BM x BN outputs per workgroup, a wave (BM / WAVES_M) x (BN / WAVES_N) of them.
// Ring of S k-steps in LDS (1 KB blocks of 8 rows x 128 bytes, 16-byte chunk c of
// row R in slot c ^ (R % 8); behind them a KB per group of 64 rows, half of it its scale
// tile). k-step kt: wait for its DMAs, barrier (which also says that every wave is
// done with k-step kt - 1), refill that slot with k-step kt + S - 1, multiply.
template <int BM, int BN, int WAVES_M, int WAVES_N, int S, int EPI>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N) void fp4_tile(Fp4Args p) {
  constexpr int BK = 128, NWAVES = WAVES_M * WAVES_N;
  constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, FM = WM / 16, FN = WN / 16;
  constexpr int A_BYTES = BM * BK, SCALES = (BM + BN) * BK, GA = BM / 64, GB = BN / 64;
  constexpr int SLOT = SCALES + (GA + GB) * 1024;
  constexpr int BLOCKS = (BM + BN) / 8, LOADS = BLOCKS / NWAVES;
  static_assert(BM % 64 == 0 && BN % 64 == 0 && BLOCKS % NWAVES == 0 && S >= 2, "tile shape");
  static_assert((FM == 2 || FM == 4) && (FN == 2 || FN == 4) && GA + GB <= NWAVES, "scale words and DMAs");
  constexpr int STAGE = WM * (2 * WN + 16);
  __shared__ __attribute__((aligned(1024))) char smem[S * SLOT > NWAVES * STAGE ? S * SLOT : NWAVES * STAGE];
  int tm, tn;
  tile_coords(p, (int)blockIdx.x, tm, tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / WAVES_N, wn = wave % WAVES_N;
  const int64_t K = p.kb;
  const int KT = p.col_tiles;
  const int64_t rows_a = min((int64_t)BM, p.m - m0), rows_b = min((int64_t)BN, p.n - n0);
  const __amdgpu_buffer_rsrc_t ra = row_rsrc(p.a + m0 * K, rows_a * K), rb = row_rsrc(p.b + n0 * K, rows_b * K);
  // Wave g < GA + GB loads the scale tiles of group g (A's, then B's) with half its lanes;
  // those of a group past the operand's rows lie past the buffer's end and read as zero.
  const int group = wave < GA ? wave : wave - GA;
  const int64_t groups = ((wave < GA ? rows_a : rows_b) + 63) >> 6;
  const __amdgpu_buffer_rsrc_t rs = row_rsrc((wave < GA ? p.as + (m0 >> 6) * KT * 512 : p.bs + (n0 >> 6) * KT * 512),
                                             groups * KT * 512);
  const uint32_t soff = lane < 32 ? (uint32_t)(group * KT * 512 + lane * 16) : 0x80000000u;

  const int drow = lane >> 3;
  const int dchunk = ((lane & 7) ^ drow) * 16;
  // Past the last column of a row the lane asks for an offset past the buffer.
  auto issue = [&](int kt) __attribute__((always_inline)) {
    char* slot = smem + (kt % S) * SLOT;
    const bool in = kt < KT && (int64_t)kt * BK + dchunk < K;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int blk = wave * LOADS + i;
      const bool is_a = blk < BM / 8;
      const int row = (is_a ? blk : blk - BM / 8) * 8 + drow;
      const uint32_t off = in ? (uint32_t)(row * K + kt * BK + dchunk) : 0x80000000u;
      dma16(is_a ? ra : rb, slot + blk * 1024, off, 0);
    }
    if (wave < GA + GB) dma16(rs, slot + SCALES + wave * 1024, soff, (kt < KT ? kt : KT - 1) * 512);
  };
  const int r16 = lane & 15;
  const int rd_row = (r16 >> 3) * 1024 + (r16 & 7) * 128;
  auto frag = [&](const char* base, int f, int h) __attribute__((always_inline)) -> v4i {
    return *reinterpret_cast<const v4i*>(base + f * 2048 + rd_row + (((lane >> 4) + 4 * h) ^ (r16 & 7)) * 16);
  };

  v4f acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < S - 1; ++t) issue(t);
  static_assert((S - 2) * (LOADS + 1) <= 63, "vmcnt range");
#pragma unroll 1
  for (int kt = 0; kt < KT; ++kt) {
    // In flight: the DMAs of k-steps kt .. kt + S - 2, oldest first.
    if (wave < GA + GB) __builtin_amdgcn_s_waitcnt(0x70 | 0xf00 | vm((S - 2) * (LOADS + 1)));
    else __builtin_amdgcn_s_waitcnt(0x70 | 0xf00 | vm((S - 2) * LOADS));
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    issue(kt + S - 1);
    __builtin_amdgcn_sched_barrier(0);
    const char* const slot = smem + (kt % S) * SLOT;
    // Byte 2 * (f % 2) + h of word f / 2 is fragment f's scale, half h.
    uint32_t sa[FM / 2], sb[FN / 2];
#pragma unroll
    for (int f = 0; f < FM / 2; ++f) {
      const int row = wm * WM + 32 * f;
      sa[f] = *reinterpret_cast<const uint32_t*>(slot + SCALES + (row >> 6) * 1024 + lane * 8 + (row >> 3 & 4));
    }
#pragma unroll
    for (int f = 0; f < FN / 2; ++f) {
      const int row = wn * WN + 32 * f;
      sb[f] = *reinterpret_cast<const uint32_t*>(slot + SCALES + (GA + (row >> 6)) * 1024 + lane * 8 + (row >> 3 & 4));
    }
    each<2>([&](auto hh) __attribute__((always_inline)) {
      constexpr int h = decltype(hh)::value;
      v4i a[FM], w[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) w[j] = frag(slot + A_BYTES, wn * FN + j, h);
#pragma unroll
      for (int i = 0; i < FM; ++i) a[i] = frag(slot, wm * FM + i, h);
      each<FM>([&](auto ii) __attribute__((always_inline)) {
        constexpr int i = decltype(ii)::value;
        each<FN>([&](auto jj) __attribute__((always_inline)) {
          constexpr int j = decltype(jj)::value;
          acc[i][j] = mfma_fp4<2 * (j & 1) + h, 2 * (i & 1) + h>(w[j], a[i], acc[i][j], sb[j >> 1], sa[i >> 1]);
        });
      });
    });
  }
  __builtin_amdgcn_s_waitcnt(0x70 | 0xf00);  // vmcnt(0): the trailing DMAs have landed
  __syncthreads();
  if (p.staged) store_staged<FM, FN, EPI>(p, acc, smem + wave * STAGE, m0 + wm * WM, n0 + wn * WN, lane);
  else store_direct<FM, FN, EPI>(p, acc, m0 + wm * WM, n0 + wn * WN, lane);
}

// ------------------------------------------------------ ping-pong kernel ----
// K % 256 == 0, staged outputs. Eight waves, 2 x 4; those of the upper half of the rows (one per
// SIMD) and of the lower half (the SIMD's other wave) take turns: while one group
// issues nothing but the matrix instructions of its k-step, from registers, the
// other reads its next fragments from LDS and issues DMAs and scale loads, with a
// barrier between the phases. Phase 2k: group 0 reads k-step k, group 1 multiplies
// k - 1; phase 2k + 1: the other way round.
//
// A k-steps live in NA = 3 LDS slots, W k-steps in NB = 2. Group 0 refills A: k-step
// k + 2 in its memory phase of k, into the slot of k - 1, and waits for k + 1 at the
// end of its compute phase. Group 1 refills W: k-step k + 2 into the slot of k, once
// its own reads of it are done (a wave's DMAs write the rows that it alone of its
// group reads; group 0 has read them a phase earlier), and waits for k + 1 before
// the barrier that publishes both to group 0. Loads past the last k-step repeat it,
// into slots that are not read again, so that the wait counts stay fixed.
// Scales of k-step k + 1 are loaded in the memory phase of k, into the other of two
// register sets; the loop takes two k-steps per trip so that no set is copied.
//
// Measured: 5.0 PFLOP/s in the loop (4096 x 4096 x 65536: 450-461 us). Matrix
// instructions on random codes from registers alone reach 6.9 to 7.4 (9.6 on zeros:
// the chip's power bounds them); without its scale loads the loop takes 430 us, without
// DMAs 383, without LDS reads 413. With starts and ends of tiles 4.3 to 4.4 PFLOP/s (12605 x
// 28672 x 5376: 877-902 us, of which storing 723 MB costs 100: a tile's registers are
// all in use, so that the next tile cannot start under its end; starting the CUs at
// different times, 904 us, does not spread that). One workgroup looping over tiles
// with the next one's loads in flight spilled and was slower.
template <int BM, int BN, int EPI>
__global__ __launch_bounds__(512) void fp4_pingpong(Fp4Args p) {
  constexpr int BK = 128, NA = 3, NB = 2;
  constexpr int WM = BM / 2, WN = BN / 4, FM = WM / 16, FN = WN / 16;
  constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK, RING = NA * A_BYTES + NB * B_BYTES;
  constexpr int PA = BM / 32, PB = BN / 32;   // 1 KB DMAs per wave and k-step
  constexpr int STAGE = WM * (2 * WN + 16);
  typedef Scales<FM, (WM % 64 == 0 ? 64 : (WM % 32 == 0 ? 32 : 16))> SA;
  typedef Scales<FN, 64> SB;
  constexpr int SL = SA::kLoads + SB::kLoads;   // scale loads per k-step
  __shared__ __attribute__((aligned(1024))) char smem[RING > 8 * STAGE ? RING : 8 * STAGE];
  char* const a_ring = smem;
  char* const b_ring = smem + NA * A_BYTES;
  int tm, tn;
  tile_coords(p, (int)blockIdx.x, tm, tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int grp = wave >> 2, q = wave & 3;    // grp: rows, q: columns, and the quarter of the DMAs
  const int64_t K = p.kb;
  const int KT = p.col_tiles;
  const int64_t rows_a = min((int64_t)BM, p.m - m0), rows_b = min((int64_t)BN, p.n - n0);
  const __amdgpu_buffer_rsrc_t r_op =
      grp == 0 ? row_rsrc(p.a + m0 * K, rows_a * K) : row_rsrc(p.b + n0 * K, rows_b * K);
  // The scale panel of A starts at a multiple of 64 rows, arow before the tile's first.
  const int arow = (int)(m0 & 63);
  const int groups_a = (int)((arow + rows_a + 63) >> 6), groups_b = (int)((rows_b + 63) >> 6);
  const __amdgpu_buffer_rsrc_t rsa = row_rsrc(p.as + (m0 >> 6) * KT * 512, (int64_t)groups_a * KT * 512);
  const __amdgpu_buffer_rsrc_t rsb = row_rsrc(p.bs + (n0 >> 6) * KT * 512, (int64_t)groups_b * KT * 512);
  const int drow = lane >> 3;
  const int dchunk = ((lane & 7) ^ drow) * 16;
  // Offset of the wave's first DMA; the others are 8 rows apart (added where they
  // are issued: kept in registers, eight offsets make the loop spill).
  const uint32_t off0 = (uint32_t)((q * (grp == 0 ? PA : PB) * 8 + drow) * K + dchunk);
  const uint32_t rows8 = (uint32_t)(8 * K);
  auto kpos = [&](int kt) __attribute__((always_inline)) { return kt < KT ? kt : KT - 1; };
  auto dma_a = [&](int kt) __attribute__((always_inline)) {
    char* const slot = a_ring + (kt % NA) * A_BYTES + q * PA * 1024;
    uint32_t off = off0;
    asm volatile("" : "+v"(off));
#pragma unroll
    for (int i = 0; i < PA; ++i) dma16(r_op, slot + i * 1024, off + i * rows8, (uint32_t)(kpos(kt) * BK));
  };
  auto dma_b = [&](int kt) __attribute__((always_inline)) {
    char* const slot = b_ring + (kt % NB) * B_BYTES + q * PB * 1024;
    uint32_t off = off0;
    asm volatile("" : "+v"(off));
#pragma unroll
    for (int i = 0; i < PB; ++i) dma16(r_op, slot + i * 1024, off + i * rows8, (uint32_t)(kpos(kt) * BK));
  };
  const int r16 = lane & 15;
  const int rd_row = (r16 >> 3) * 1024 + (r16 & 7) * 128;
  const int rd0 = rd_row + ((lane >> 4) ^ (r16 & 7)) * 16, rd1 = rd_row + (((lane >> 4) + 4) ^ (r16 & 7)) * 16;
  v4f acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  v4i a0[FM], w0[FN], a1[FM], w1[FN];
  SA sa[2];
  SB sb[2];
  auto scales = [&](int kt, int set) __attribute__((always_inline)) {
    sa[set].load(rsa, groups_a, arow + grp * WM, KT, kpos(kt), lane);
    sb[set].load(rsb, groups_b, q * WN, KT, kpos(kt), lane);
  };
  auto read_all = [&](int kt) __attribute__((always_inline)) {
    const char* const pa = a_ring + (kt % NA) * A_BYTES + grp * FM * 2048;
    const char* const pb = b_ring + (kt % NB) * B_BYTES + q * FN * 2048;
#pragma unroll
    for (int i = 0; i < FM; ++i) a0[i] = *reinterpret_cast<const v4i*>(pa + i * 2048 + rd0);
#pragma unroll
    for (int j = 0; j < FN; ++j) w0[j] = *reinterpret_cast<const v4i*>(pb + j * 2048 + rd0);
#pragma unroll
    for (int i = 0; i < FM; ++i) a1[i] = *reinterpret_cast<const v4i*>(pa + i * 2048 + rd1);
#pragma unroll
    for (int j = 0; j < FN; ++j) w1[j] = *reinterpret_cast<const v4i*>(pb + j * 2048 + rd1);
  };
  auto compute = [&](auto which) __attribute__((always_inline)) {
    constexpr int set = decltype(which)::value;
    sa[set].settle(arow + grp * WM);
    auto half = [&](const v4i (&a)[FM], const v4i (&w)[FN], auto hh) __attribute__((always_inline)) {
      constexpr int h = decltype(hh)::value;
      each<FM>([&](auto ii) __attribute__((always_inline)) {
        constexpr int i = decltype(ii)::value;
        each<FN>([&](auto jj) __attribute__((always_inline)) {
          constexpr int j = decltype(jj)::value;
          acc[i][j] = mfma_fp4<SB::byte(j, h), SA::byte(i, h)>(w[j], a[i], acc[i][j], sb[set].w[j >> 1],
                                                               sa[set].w[i >> 1]);
        });
      });
    };
    half(a0, w0, std::integral_constant<int, 0>());
    half(a1, w1, std::integral_constant<int, 1>());
  };
  auto barrier = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  typedef std::integral_constant<int, 0> Even;
  typedef std::integral_constant<int, 1> Odd;
  constexpr int kPro = 0x70 | 0xf00, kLds = 0xc07f;   // kPro | vm(n): vmcnt(n); kLds: lgkmcnt(0)
  constexpr int kA = PA + SL, kB = PB + SL;           // one k-step's loads, left in flight
  static_assert(kA <= 63 && kB <= 63, "vmcnt range");
  if (grp == 0) {
    scales(0, 0);
    __builtin_amdgcn_sched_barrier(0);
    dma_a(0);
    dma_a(1);
    __builtin_amdgcn_s_waitcnt(kPro | vm(PA));
    barrier();
    auto step = [&](int kt, auto set) __attribute__((always_inline)) {
      read_all(kt);
      scales(kt + 1, decltype(set)::value ^ 1);
      __builtin_amdgcn_sched_barrier(0);
      dma_a(kt + 2);
      __builtin_amdgcn_s_waitcnt(kLds);
      barrier();
      compute(set);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(kPro | vm(kA));  // A(kt + 1) landed
      barrier();
    };
    int kt = 0;
#pragma unroll 1
    for (; kt + 1 < KT; kt += 2) {
      step(kt, Even());
      step(kt + 1, Odd());
    }
    if (kt < KT) step(kt, Even());
    barrier();
  } else {
    scales(0, 0);
    __builtin_amdgcn_sched_barrier(0);
    dma_b(0);
    dma_b(1);
    __builtin_amdgcn_s_waitcnt(kPro | vm(PB));
    barrier();
    barrier();
    auto step = [&](int kt, auto set) __attribute__((always_inline)) {
      read_all(kt);
      __builtin_amdgcn_s_waitcnt(kLds);
      __builtin_amdgcn_sched_barrier(0);
      dma_b(kt + 2);
      __builtin_amdgcn_sched_barrier(0);
      scales(kt + 1, decltype(set)::value ^ 1);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(kPro | vm(kB));  // W(kt + 1) landed
      barrier();
      compute(set);
      barrier();
    };
    int kt = 0;
#pragma unroll 1
    for (; kt + 1 < KT; kt += 2) {
      step(kt, Even());
      step(kt + 1, Odd());
    }
    if (kt < KT) step(kt, Even());
  }
  __builtin_amdgcn_s_waitcnt(kPro);  // the trailing DMAs have landed
  __syncthreads();
  store_staged<FM, FN, EPI>(p, acc, smem + wave * STAGE, m0 + grp * WM, n0 + q * WN, lane);
}

template <int BM, int BN>
int launch_pingpong(Fp4Args p, int epilogue, hipStream_t s) {
  const int64_t tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
  LR_REQUIRE(p.kb % 128 == 0 && p.staged, "mxfp4_gemm: not a shape of the ping-pong kernel");
  LR_REQUIRE(tm * tn <= kMaxBlocks / 2, "mxfp4_gemm: %lld output tiles are not supported", (long long)(tm * tn));
  p.tiles_m = (int)tm;
  p.tiles_n = (int)tn;
  const dim3 grid((unsigned)(tm * tn));
  if (epilogue == EPI_BF16) fp4_pingpong<BM, BN, EPI_BF16><<<grid, 512, 0, s>>>(p);
  else if (epilogue == EPI_GELU) fp4_pingpong<BM, BN, EPI_GELU><<<grid, 512, 0, s>>>(p);
  else fp4_pingpong<BM, BN, EPI_GATED><<<grid, 512, 0, s>>>(p);
  return check_launch("mxfp4_gemm");
}

// --------------------------------------------------------- few rows kernel ----
// The waves' sums of (16 * FM) x (16 * FN) outputs, joined in wave order through LDS
// (wave w's at sums + w * pitch), and the epilogue.
template <int FM, int FN, int WAVES, int EPI>
__device__ __forceinline__ void store_few(const Fp4Args& p, const v4f (&acc)[FM][FN], char* sums, int pitch,
                                          int64_t m0, int64_t n0) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r16 = lane & 15, lg = lane >> 4;
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) *reinterpret_cast<v4f*>(sums + wave * pitch + (i * FN + j) * 1024 + lane * 16) = acc[i][j];
  __syncthreads();
  for (int t = threadIdx.x >> 6; t < FM * FN; t += WAVES) {
    v4f v = *reinterpret_cast<const v4f*>(sums + t * 1024 + lane * 16);
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += *reinterpret_cast<const v4f*>(sums + w * pitch + t * 1024 + lane * 16);
    const int64_t row = m0 + 16 * (t / FN) + r16, col = n0 + 16 * (t % FN) + 4 * lg;
    if (row >= p.m) continue;
    if (!p.staged) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < p.n) store_scalar<EPI>(p, row, col + e, v[e]);
      continue;
    }
    if (col >= p.n) continue;
    const int64_t o = row * p.n + col;
    const uint2 b = p.bias ? *reinterpret_cast<const uint2*>(p.bias + col) : make_uint2(0u, 0u);
    uint2 x = make_uint2(0u, 0u), g = x;
    if (EPI == EPI_GATED) {
      x = *reinterpret_cast<const uint2*>(p.resid + o);
      g = *reinterpret_cast<const uint2*>(p.table + table_row(p, row) * p.table_width + (int64_t)p.gate_slot * p.n +
                                          col);
    }
    const float y0 = finish<EPI>(round_bf(v[0] + bf_lo(b.x)), bf_lo(g.x), bf_lo(x.x));
    const float y1 = finish<EPI>(round_bf(v[1] + bf_hi(b.x)), bf_hi(g.x), bf_hi(x.x));
    const float y2 = finish<EPI>(round_bf(v[2] + bf_lo(b.y)), bf_lo(g.y), bf_lo(x.y));
    const float y3 = finish<EPI>(round_bf(v[3] + bf_hi(b.y)), bf_hi(g.y), bf_hi(x.y));
    *reinterpret_cast<uint2*>(p.c + o) = make_uint2(pack_bf2(y0, y1), pack_bf2(y2, y3));
  }
}

// At most 16 * FM rows: what counts is the stream of weights. A workgroup has 16 * FN
// columns; its WAVES waves take every WAVES-th k-step each and add their sums in wave
// order at the end. A wave is on its own until then: it keeps the next S - 1 of its
// k-steps in flight into a ring of LDS that no other wave touches, so that it meets
// no barrier, with whole 128-byte lines of both operands and their scales (fragments
// straight into registers read half lines, and their waits, which count in issue
// order, would hold up the ring). 1 x 21504 x 5376: 12.0 us, 5.1 TB/s of weights that partly
// come out of the caches, 13.2 us, 4.6 TB/s, where none do; 16 x 5376 x 14336: 9.1 us, 4.5.
template <int FM, int FN, int WAVES, int S, int EPI>
__global__ __launch_bounds__(64 * WAVES) void fp4_few(Fp4Args p) {
  constexpr int BK = 128;
  constexpr int W_AT = FM * 2048, SA_AT = W_AT + FN * 2048, SB_AT = SA_AT + 256, SLOT = SB_AT + 256;
  constexpr int LOADS = 2 * FM + 2 * FN + 2;   // per k-step
  static_assert(FM <= 2 && FN <= 2 && (S - 2) * LOADS <= 63, "one scale word per lane and operand; ring");
  static_assert(FM * FN * 1024 <= S * SLOT, "the sums fit the ring");
  __shared__ __attribute__((aligned(1024))) char smem[WAVES][S * SLOT];
  const int64_t n0 = (int64_t)blockIdx.x * (16 * FN), m0 = (int64_t)blockIdx.y * (16 * FM);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  char* const ring = smem[wave];
  const int r16 = lane & 15, lg = lane >> 4;
  const int64_t K = p.kb;
  const int KT = p.col_tiles;
  const int mine = KT > wave ? (KT - wave + WAVES - 1) / WAVES : 0;   // this wave's k-steps
  const int64_t rows_a = min((int64_t)(16 * FM), p.m - m0), rows_b = min((int64_t)(16 * FN), p.n - n0);
  const __amdgpu_buffer_rsrc_t ra = row_rsrc(p.a + m0 * K, rows_a * K), rb = row_rsrc(p.b + n0 * K, rows_b * K);
  const __amdgpu_buffer_rsrc_t rsa = row_rsrc(p.as + (m0 >> 6) * KT * 512, (int64_t)KT * 512);
  const __amdgpu_buffer_rsrc_t rsb = row_rsrc(p.bs + (n0 >> 6) * KT * 512, (int64_t)KT * 512);
  // As in the tile kernels: 1 KB blocks of 8 rows, chunk c of row R in slot c ^ (R % 8).
  const int drow = lane >> 3, dchunk = ((lane & 7) ^ drow) * 16;
  const uint32_t off0 = (uint32_t)(drow * K + dchunk), rows8 = (uint32_t)(8 * K);
  const int end = (int)K - dchunk;
  // Two fragments' scale bytes per lane: those of the pair of 16 rows that holds the wave's.
  const uint32_t sa_off = lane * 8 + ((uint32_t)m0 & 32) / 8, sb_off = lane * 8 + ((uint32_t)n0 & 32) / 8;
  auto issue = [&](int i) __attribute__((always_inline)) {
    const int kt = wave + min(i, mine - 1) * WAVES;
    char* const slot = ring + i % S * SLOT;
    const uint32_t past = kt * BK < end ? 0u : 0x80000000u;   // a row's end: reads as zero
    const int soff = kt * BK;
#pragma unroll
    for (int j = 0; j < 2 * FN; ++j) dma16(rb, slot + W_AT + j * 1024, (off0 + j * rows8) | past, soff);
#pragma unroll
    for (int j = 0; j < 2 * FM; ++j) dma16(ra, slot + j * 1024, (off0 + j * rows8) | past, soff);
    dma4(rsa, slot + SA_AT, sa_off, kt * 512);
    dma4(rsb, slot + SB_AT, sb_off, kt * 512);
  };
  v4f acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  if (mine > 0) {
    const int rd_row = (r16 >> 3) * 1024 + (r16 & 7) * 128;
    const int rd0 = rd_row + (lg ^ (r16 & 7)) * 16, rd1 = rd_row + ((lg + 4) ^ (r16 & 7)) * 16;
    // A single fragment may be the upper one of its pair.
    const int sh_a = FM == 1 ? (int)(m0 & 16) : 0, sh_b = FN == 1 ? (int)(n0 & 16) : 0;
#pragma unroll
    for (int i = 0; i < S - 1; ++i) issue(i);
#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
      constexpr int kVm = (S - 2) * LOADS;
      __builtin_amdgcn_s_waitcnt(0x70 | 0xf00 | vm(kVm));   // k-step i has landed
      asm volatile("" ::: "memory");
      const char* const slot = ring + i % S * SLOT;
      v4i a[2][FM], w[2][FN];
#pragma unroll
      for (int f = 0; f < FM; ++f) {
        a[0][f] = *reinterpret_cast<const v4i*>(slot + f * 2048 + rd0);
        a[1][f] = *reinterpret_cast<const v4i*>(slot + f * 2048 + rd1);
      }
#pragma unroll
      for (int f = 0; f < FN; ++f) {
        w[0][f] = *reinterpret_cast<const v4i*>(slot + W_AT + f * 2048 + rd0);
        w[1][f] = *reinterpret_cast<const v4i*>(slot + W_AT + f * 2048 + rd1);
      }
      const uint32_t sa = *reinterpret_cast<const uint32_t*>(slot + SA_AT + lane * 4) >> sh_a;
      const uint32_t sb = *reinterpret_cast<const uint32_t*>(slot + SB_AT + lane * 4) >> sh_b;
      // The slot of k-step i - 1 is free: its reads were waited for by its products.
      issue(i + S - 1);
      each<2>([&](auto hh) __attribute__((always_inline)) {
        constexpr int h = decltype(hh)::value;
        each<FM>([&](auto ii) __attribute__((always_inline)) {
          constexpr int f = decltype(ii)::value;
          each<FN>([&](auto jj) __attribute__((always_inline)) {
            constexpr int j = decltype(jj)::value;
            acc[f][j] = mfma_fp4<2 * j + h, 2 * f + h>(w[h][j], a[h][f], acc[f][j], sb, sa);
          });
        });
      });
    }
    __builtin_amdgcn_s_waitcnt(0x70 | 0xf00);  // vmcnt(0): the trailing DMAs have landed
    asm volatile("" ::: "memory");
  }
  store_few<FM, FN, WAVES, EPI>(p, acc, smem[0], S * SLOT, m0, n0);
}

// One row, quantized by every workgroup for itself, which costs less than a kernel
// before this one: fp4_few with the row's codes and scales in LDS, each wave those of
// its own k-steps. The first weights are in flight meanwhile. Against the two kernels,
// back to back: 1 x 21504 x 5376 14.1-14.6 us (15.4), 4.2 TB/s of weights, 1 x 5120 x 5120 6.3 (7.3), 1 x 15360 x
// 5120 9.9 (12.1); and the host launches one kernel, 10 us a call for 13. The
// quantizing takes every wave 50 instructions per 512 columns, so that from some 7000 on
// it costs more than its kernel: 1 x 5120 x 20480 18.1 us (17.2), 1 x 5376 x 14336 11.6 (11.1).
constexpr int kTokenPairs = 12, kTokenK = 512 * kTokenPairs;   // pairs of k-steps and columns per wave
template <int DTYPE, int FN, int WAVES, int S, int EPI>
__global__ __launch_bounds__(64 * WAVES) void fp4_token(Fp4Args p, const char* x, int64_t width) {
  constexpr int BK = 128, SB_AT = FN * 2048, SLOT = SB_AT + 256, LOADS = 2 * FN + 1;
  static_assert(FN <= 2 && (S - 2) * LOADS <= 63 && FN * 1024 <= S * SLOT, "ring");
  // One object: between two the compiler would wait for all DMAs before every read.
  constexpr int RINGS = WAVES * S * SLOT, CODES = WAVES * kTokenK / 2;
  __shared__ __attribute__((aligned(1024))) char smem[RINGS + CODES + CODES / 16];
  char* const codes = smem + RINGS;
  char* const scales = codes + CODES;
  typedef Row8<DTYPE> R;
  const int64_t n0 = (int64_t)blockIdx.x * (16 * FN);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  char* const ring = smem + wave * (S * SLOT);
  const int r16 = lane & 15, lg = lane >> 4;
  const int64_t K = p.kb;
  const int KT = p.col_tiles;
  const int mine = KT > wave ? (KT - wave + WAVES - 1) / WAVES : 0;   // this wave's k-steps
  const int64_t rows_b = min((int64_t)(16 * FN), p.n - n0);
  const __amdgpu_buffer_rsrc_t rb = row_rsrc(p.b + n0 * K, rows_b * K);
  const __amdgpu_buffer_rsrc_t rsb = row_rsrc(p.bs + (n0 >> 6) * KT * 512, (int64_t)KT * 512);
  const __amdgpu_buffer_rsrc_t rx = row_rsrc(x, width * R::kBytes);
  const int drow = lane >> 3, dchunk = ((lane & 7) ^ drow) * 16;
  const uint32_t off0 = (uint32_t)(drow * K + dchunk), rows8 = (uint32_t)(8 * K);
  const int end = (int)K - dchunk;
  const uint32_t sb_off = lane * 8 + ((uint32_t)n0 & 32) / 8;
  auto issue = [&](int i) __attribute__((always_inline)) {
    const int kt = wave + min(i, mine - 1) * WAVES;
    char* const slot = ring + i % S * SLOT;
    const uint32_t past = kt * BK < end ? 0u : 0x80000000u;   // a row's end: reads as zero
#pragma unroll
    for (int j = 0; j < 2 * FN; ++j) dma16(rb, slot + j * 1024, (off0 + j * rows8) | past, kt * BK);
    dma4(rsb, slot + SB_AT, sb_off, kt * 512);
  };
  v4f acc[1][FN];
#pragma unroll
  for (int j = 0; j < FN; ++j) acc[0][j] = v4f{0.f, 0.f, 0.f, 0.f};
  if (mine > 0) {
    // Half a wave per k-step, eight values per lane.
    const int chunk = lane & 31;
    R v[kTokenPairs];
#pragma unroll
    for (int u = 0; u < kTokenPairs; ++u) {
      const int i = 2 * u + (lane >> 5);
      // Past the row's end (width % 8 == 0) or the wave's k-steps: zeros.
      v[u].load(rx, i < mine ? (uint32_t)((wave + i * WAVES) * 256 + chunk * 8) * R::kBytes : 0x80000000u);
    }
#pragma unroll
    for (int i = 0; i < S - 1; ++i) issue(i);
#pragma unroll
    for (int u = 0; u < kTokenPairs; ++u) {
      const int i = 2 * u + (lane >> 5), kt = wave + i * WAVES;
      const uint32_t byte = scale_byte(quad_max(v[u].magnitude()));
      if (i >= mine) continue;
      // 2^e as fp32 is the byte in the exponent field; e = -127 is a subnormal.
      const float scale = __uint_as_float(byte == 0 ? 0x00400000u : byte << 23);
      *reinterpret_cast<uint32_t*>(codes + kt * BK + chunk * 4) = byte == 255 ? 0u : v[u].codes(scale);
      if ((lane & 3) == 0) scales[kt * 8 + (chunk >> 2)] = (char)byte;
    }
    // The wave reads what it wrote itself: LDS operations of a wave stay in order.
    asm volatile("" ::: "memory");
    const int rd_row = (r16 >> 3) * 1024 + (r16 & 7) * 128;
    const int rd0 = rd_row + (lg ^ (r16 & 7)) * 16, rd1 = rd_row + ((lg + 4) ^ (r16 & 7)) * 16;
    const int sh_b = FN == 1 ? (int)(n0 & 16) : 0;
#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
      constexpr int kVm = (S - 2) * LOADS;
      __builtin_amdgcn_s_waitcnt(0x70 | 0xf00 | vm(kVm));   // k-step i has landed
      asm volatile("" ::: "memory");
      const char* const slot = ring + i % S * SLOT;
      const int kt = wave + i * WAVES;
      // The row in all 16 of the fragment's: the others' outputs are not stored.
      v4i a[2], w[2][FN];
#pragma unroll
      for (int h = 0; h < 2; ++h) a[h] = *reinterpret_cast<const v4i*>(codes + kt * BK + 64 * h + 16 * lg);
      const uint32_t sa = (uint8_t)scales[kt * 8 + lg] | (uint32_t)(uint8_t)scales[kt * 8 + 4 + lg] << 8;
#pragma unroll
      for (int f = 0; f < FN; ++f) {
        w[0][f] = *reinterpret_cast<const v4i*>(slot + f * 2048 + rd0);
        w[1][f] = *reinterpret_cast<const v4i*>(slot + f * 2048 + rd1);
      }
      const uint32_t sb = *reinterpret_cast<const uint32_t*>(slot + SB_AT + lane * 4) >> sh_b;
      // The slot of k-step i - 1 is free: its reads were waited for by its products.
      issue(i + S - 1);
      each<2>([&](auto hh) __attribute__((always_inline)) {
        constexpr int h = decltype(hh)::value;
        each<FN>([&](auto jj) __attribute__((always_inline)) {
          constexpr int j = decltype(jj)::value;
          acc[0][j] = mfma_fp4<2 * j + h, h>(w[h][j], a[h], acc[0][j], sb, sa);
        });
      });
    }
    __builtin_amdgcn_s_waitcnt(0x70 | 0xf00);  // vmcnt(0): the trailing DMAs have landed
    asm volatile("" ::: "memory");
  }
  store_few<1, FN, WAVES, EPI>(p, acc, smem, S * SLOT, 0, n0);
}

template <int FM, int FN, int WAVES, int S>
int launch_few(const Fp4Args& p, int epilogue, hipStream_t s) {
  const int64_t gx = (p.n + 16 * FN - 1) / (16 * FN), gy = (p.m + 16 * FM - 1) / (16 * FM);
  LR_REQUIRE(gx <= kMaxBlocks && gy <= 65535, "mxfp4_gemm: m=%lld, n=%lld are not supported", (long long)p.m,
             (long long)p.n);
  const dim3 grid((unsigned)gx, (unsigned)gy);
  if (epilogue == EPI_BF16) fp4_few<FM, FN, WAVES, S, EPI_BF16><<<grid, 64 * WAVES, 0, s>>>(p);
  else if (epilogue == EPI_GELU) fp4_few<FM, FN, WAVES, S, EPI_GELU><<<grid, 64 * WAVES, 0, s>>>(p);
  else fp4_few<FM, FN, WAVES, S, EPI_GATED><<<grid, 64 * WAVES, 0, s>>>(p);
  return check_launch("mxfp4_gemm");
}

template <int DTYPE, int WAVES>
int launch_token_waves(const Fp4Args& p, const char* x, int64_t width, int epilogue, hipStream_t s) {
  const dim3 grid((unsigned)((p.n + 31) / 32));
  if (epilogue == EPI_BF16) fp4_token<DTYPE, 2, WAVES, 5, EPI_BF16><<<grid, 64 * WAVES, 0, s>>>(p, x, width);
  else if (epilogue == EPI_GELU) fp4_token<DTYPE, 2, WAVES, 5, EPI_GELU><<<grid, 64 * WAVES, 0, s>>>(p, x, width);
  else fp4_token<DTYPE, 2, WAVES, 5, EPI_GATED><<<grid, 64 * WAVES, 0, s>>>(p, x, width);
  return check_launch("mxfp4_linear");
}

template <int DTYPE>
int launch_token(const Fp4Args& p, const void* x, int64_t width, bool two, int epilogue, hipStream_t s) {
  const char* const px = static_cast<const char*>(x);
  return two ? launch_token_waves<DTYPE, 2>(p, px, width, epilogue, s)
             : launch_token_waves<DTYPE, 1>(p, px, width, epilogue, s);
}

template <int BM, int BN, int WAVES_M, int WAVES_N, int S>
int launch_tile(Fp4Args p, int epilogue, hipStream_t s) {
  const int64_t tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
  LR_REQUIRE(tm * tn <= kMaxBlocks, "mxfp4_gemm: %lld output tiles are not supported", (long long)(tm * tn));
  p.tiles_m = (int)tm;
  p.tiles_n = (int)tn;
  const dim3 grid((unsigned)(tm * tn)), block(64 * WAVES_M * WAVES_N);
  if (epilogue == EPI_BF16) fp4_tile<BM, BN, WAVES_M, WAVES_N, S, EPI_BF16><<<grid, block, 0, s>>>(p);
  else if (epilogue == EPI_GELU) fp4_tile<BM, BN, WAVES_M, WAVES_N, S, EPI_GELU><<<grid, block, 0, s>>>(p);
  else fp4_tile<BM, BN, WAVES_M, WAVES_N, S, EPI_GATED><<<grid, block, 0, s>>>(p);
  return check_launch("mxfp4_gemm");
}

// -------------------------------------------------------------- schedule ----
// The ping-pong kernel's tiles, and what one costs: us of a k-step and of a tile's
// start and end, for the 256 CUs' tiles together, from 990 timings (six tiles, 165
// shapes, M 72 to 12605, N 2048 to 28672, K 1024 to 20480; mean error 5% beside 3 us per
// call). The choice that it makes is on average 0.1% and at most 7% slower than the
// fastest tile of those shapes.
struct Tile {
  int rows, cols;
  double factor;
  int (*run)(Fp4Args, int, hipStream_t);
};
const Tile kTiles[] = {
    {256, 256, 1.113, launch_pingpong<256, 256>}, {192, 256, 1.144, launch_pingpong<192, 256>},
    {160, 256, 1.202, launch_pingpong<160, 256>}, {128, 256, 1.162, launch_pingpong<128, 256>},
    {128, 128, 0.985, launch_pingpong<128, 128>}, {64, 128, 0.872, launch_pingpong<64, 128>},
};

double tile_us(const Tile& t, int64_t m, int64_t n, int64_t ksteps, int64_t cus) {
  const int64_t tiles = ((m + t.rows - 1) / t.rows) * ((n + t.cols - 1) / t.cols);
  const int64_t full = tiles / cus, rest = tiles % cus;
  // A last round with few tiles is nearly half as long: the chip's power is theirs.
  const double rounds = (double)full + (rest ? 0.598 + 0.402 * (double)rest / (double)cus : 0.0);
  const double size = t.rows * t.cols / 65536.0;
  return rounds * ((double)ksteps * (0.378 + 1.291 * size) * t.factor + 0.148 + 5.867 * size);
}

int launch(const Fp4Args& p, int epilogue, hipStream_t s) {
  const int64_t cus = compute_units();
  // Few rows: while all its workgroups are resident (four of one wave's ring per CU,
  // two of two waves'), the kernel that streams the weights. Measured at 1 to 256 rows
  // and 13 weights: up to 3.4 times faster than the best tile (1 row, K = 20480, N =
  // 5120: 14 against 47 us), level at 900 to 1000 workgroups, 1.3 to 3.5 times slower
  // above 1280. Two waves from 512 workgroups down: 8.8 against 11.9 us at 1 row, K =
  // 14336, N = 5376; at 672 they no longer fit (16.6 against 13.0 us, N = 21504).
  const int rows = p.m <= 16 ? 16 : 32;
  const int64_t few = (p.n + 31) / 32 * ((p.m + rows - 1) / rows);
  if (few <= 4 * cus) {
    if (rows == 16) return few <= 2 * cus ? launch_few<1, 2, 2, 5>(p, epilogue, s) : launch_few<1, 2, 1, 5>(p, epilogue, s);
    return few <= 2 * cus ? launch_few<2, 2, 2, 4>(p, epilogue, s) : launch_few<2, 2, 1, 4>(p, epilogue, s);
  }
  // 64 x 128 tiles of one round: five k-steps in flight count more than matrix units that
  // never pause (the ping-pong kernel has two): 256 x 5120 x 5120 12.3 us for 13.2, 64 x 21504 x
  // 5376 14.5 for 16.2, 256 x 5120 x 20480 39 for 46; in two rounds 24.7 for 19.9 (128 x 20480 x
  // 5120). And for 18.3, 22.0 and 77 of the 128 x 128 tiles.
  const bool one_round = (p.m + 63) / 64 * ((p.n + 127) / 128) <= cus;
  // The ping-pong kernel takes whole k-steps and whole-line stores only.
  if (p.kb % 128 || !p.staged)
    return one_round ? launch_tile<64, 128, 2, 4, 5>(p, epilogue, s) : launch_tile<128, 128, 2, 2, 2>(p, epilogue, s);
  const Tile* best = nullptr;
  double us = 0.0;
  for (const Tile& t : kTiles) {
    const double e = tile_us(t, p.m, p.n, p.col_tiles, cus);
    if (!best || e < us) {
      best = &t;
      us = e;
    }
  }
  if (best->rows == 64 && one_round) return launch_tile<64, 128, 2, 4, 5>(p, epilogue, s);
  return best->run(p, epilogue, s);
}

// Checks a product's arguments and fills p with them; p.m stays 0 where there is nothing to do.
int fill(Fp4Args& p, const void* a, const void* a_scale, const void* b, const void* b_scale, int64_t m, int64_t n,
         int64_t k, const void* bias, void* out, int epilogue, const void* residual, const void* table,
         int64_t table_rows, int64_t table_width, const int64_t* indices, int64_t sequence, int gate_slot) {
  LR_REQUIRE(epilogue == EPI_BF16 || epilogue == EPI_GELU || epilogue == EPI_GATED,
             "mxfp4_gemm: unknown epilogue %d", epilogue);
  LR_REQUIRE(m >= 0 && n >= 0 && k >= 0, "mxfp4_gemm: negative shape m=%lld n=%lld k=%lld", (long long)m,
             (long long)n, (long long)k);
  if (m == 0 || n == 0) return LR_OK;
  LR_REQUIRE(k > 0 && k <= (1LL << 23), "mxfp4_gemm: k=%lld must lie in [1, 2^23]", (long long)k);
  LR_REQUIRE(m <= (1LL << 31) && n <= (1LL << 31), "mxfp4_gemm: m=%lld, n=%lld are not supported", (long long)m,
             (long long)n);
  LR_REQUIRE(a && a_scale && b && b_scale && out, "mxfp4_gemm: null pointer");
  LR_REQUIRE(aligned(a, 16) && aligned(a_scale, 16) && aligned(b, 16) && aligned(b_scale, 16) && aligned(out, 2),
             "mxfp4_gemm: codes and scales must be 16-byte aligned");
  if (epilogue == EPI_GATED) {
    LR_REQUIRE(residual && table && indices, "mxfp4_gemm: the gated residual needs residual, table and indices");
    LR_REQUIRE(sequence > 0 && table_rows > 0, "mxfp4_gemm: empty sequence or table");
    LR_REQUIRE(gate_slot >= 0 && ((int64_t)gate_slot + 1) * n <= table_width,
               "mxfp4_gemm: gate slot %d of width %lld lies past a table row of %lld", gate_slot, (long long)n,
               (long long)table_width);
  }
  p.a = static_cast<const uint8_t*>(a);
  p.as = static_cast<const uint8_t*>(a_scale);
  p.b = static_cast<const uint8_t*>(b);
  p.bs = static_cast<const uint8_t*>(b_scale);
  p.bias = static_cast<const uint16_t*>(bias);
  p.c = static_cast<uint16_t*>(out);
  p.resid = static_cast<const uint16_t*>(residual);
  p.table = static_cast<const uint16_t*>(table);
  p.indices = indices;
  p.m = m;
  p.n = n;
  p.kb = (k + 31) / 32 * 16;
  p.col_tiles = (int)mxfp4_scale_tiles(k);
  p.table_rows = table_rows;
  p.table_width = table_width;
  p.sequence = sequence;
  p.gate_slot = gate_slot;
  p.staged = n % 8 == 0 && aligned(out, 16) && (!bias || aligned(bias, 8)) &&
             (epilogue != EPI_GATED || (aligned(residual, 16) && aligned(table, 16) && table_width % 8 == 0));
  return LR_OK;
}

}  // namespace
}  // namespace lr

using namespace lr;

extern "C" int lr_mxfp4_gemm(const void* a, const void* a_scale, const void* b, const void* b_scale, int64_t m,
                             int64_t n, int64_t k, const void* bias, void* out, int epilogue, const void* residual,
                             const void* table, int64_t table_rows, int64_t table_width, const int64_t* indices,
                             int64_t sequence, int gate_slot, void* stream) {
  Fp4Args p = {};
  if (int rc = fill(p, a, a_scale, b, b_scale, m, n, k, bias, out, epilogue, residual, table, table_rows, table_width,
                    indices, sequence, gate_slot))
    return rc;
  return p.m ? launch(p, epilogue, as_stream(stream)) : LR_OK;
}

extern "C" int lr_mxfp4_linear(const void* x, int dtype, int64_t m, int64_t n, int64_t k, void* scratch,
                               int64_t scratch_bytes, const void* b, const void* b_scale, const void* bias, void* out,
                               int epilogue, const void* residual, const void* table, int64_t table_rows,
                               int64_t table_width, const int64_t* indices, int64_t sequence, int gate_slot,
                               void* stream) {
  LR_REQUIRE(m >= 0 && n >= 0 && k > 0, "mxfp4_linear: bad shape m=%lld n=%lld k=%lld", (long long)m, (long long)n,
             (long long)k);
  const int64_t codes = (m * ((k + 31) / 32 * 16) + 255) / 256 * 256;
  const int64_t need = codes + (m + 63) / 64 * mxfp4_scale_tiles(k) * 512;
  LR_REQUIRE(m == 0 || (scratch && aligned(scratch, 16) && scratch_bytes >= need),
             "mxfp4_linear: the scratch must be 16-byte aligned and hold %lld bytes", (long long)need);
  LR_REQUIRE(dtype == LR_DTYPE_BF16 || dtype == LR_DTYPE_F16 || dtype == LR_DTYPE_F32,
             "mxfp4_linear: unknown dtype %d", dtype);
  char* const scales = static_cast<char*>(scratch) + codes;
  Fp4Args p = {};
  if (int rc = fill(p, scratch, scales, b, b_scale, m, n, k, bias, out, epilogue, residual, table, table_rows,
                    table_width, indices, sequence, gate_slot))
    return rc;
  if (p.m == 0) return LR_OK;
  hipStream_t s = as_stream(stream);
  const int64_t few = (n + 31) / 32, cus = compute_units();
  const bool two = few <= 2 * cus;   // waves, as in launch()
  if (m == 1 && few <= 4 * cus && k <= (two ? 2 : 1) * kTokenK && k % 8 == 0 && x && aligned(x, 16)) {
    if (dtype == LR_DTYPE_BF16) return launch_token<LR_DTYPE_BF16>(p, x, k, two, epilogue, s);
    if (dtype == LR_DTYPE_F16) return launch_token<LR_DTYPE_F16>(p, x, k, two, epilogue, s);
    return launch_token<LR_DTYPE_F32>(p, x, k, two, epilogue, s);
  }
  if (int rc = lr_quantize_rows_mxfp4(x, dtype, m, k, scratch, scales, stream)) return rc;
  return launch(p, epilogue, s);
}
