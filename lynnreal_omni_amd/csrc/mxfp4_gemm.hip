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
#include "lr_device.h"
#include "lr_mxfp4.h"
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
  int tiles_m, tiles_n, group_m;
  int staged;             // N % 8 == 0 and 16-byte aligned output (residual, table) rows
};

enum { EPI_BF16 = LR_EPI_BF16, EPI_GELU = LR_EPI_GELU_TANH, EPI_GATED = LR_EPI_GATED_RESIDUAL };

// One scaled MFMA; byte `wo` of ws and `ao` of as hold the lane's scales. The
// byte selects are instruction fields: after unrolling, one case is left.
template <int WO, int AO>
__device__ __forceinline__ v4f mfma_sel(const v8i& w, const v8i& a, const v4f& c, int ws, int as) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 4, 4, WO, ws, AO, as);
}
template <int WO>
__device__ __forceinline__ v4f mfma_sel_a(const v8i& w, const v8i& a, const v4f& c, int ws, int ao, int as) {
  switch (ao) {
    case 0: return mfma_sel<WO, 0>(w, a, c, ws, as);
    case 1: return mfma_sel<WO, 1>(w, a, c, ws, as);
    case 2: return mfma_sel<WO, 2>(w, a, c, ws, as);
    default: return mfma_sel<WO, 3>(w, a, c, ws, as);
  }
}
__device__ __forceinline__ v4f mfma_fp4(const v4i& w, const v4i& a, const v4f& c, int wo, int ws, int ao, int as) {
  const v8i w8 = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
  switch (wo) {
    case 0: return mfma_sel_a<0>(w8, a8, c, ws, ao, as);
    case 1: return mfma_sel_a<1>(w8, a8, c, ws, ao, as);
    case 2: return mfma_sel_a<2>(w8, a8, c, ws, ao, as);
    default: return mfma_sel_a<3>(w8, a8, c, ws, ao, as);
  }
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
// M-grouped range of tiles so that its L2 holds the panels its CUs share.
__device__ __forceinline__ void tile_coords(const Fp4Args& p, int pid, int& tm, int& tn) {
  const int total = p.tiles_m * p.tiles_n;
  const int xcd = pid & 7, local = pid >> 3;
  const int q = total >> 3, r = total & 7;
  const int lid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + local;
  const int span = p.group_m * p.tiles_n;
  const int g = lid / span;
  const int first = g * p.group_m;
  const int gm = min(p.tiles_m - first, p.group_m);
  const int within = lid - g * span;
  tm = first + within % gm;
  tn = within / gm;
}

typedef __attribute__((address_space(3))) void* lds_ptr_t;
// 16 bytes per lane from a buffer straight into LDS at lds + 16 * lane; offsets
// past the buffer's end read as zero.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rsrc, void* lds, uint32_t voffset, uint32_t soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)lds, 16, voffset, soffset, 0, 0);
}

// The scale registers of 16 * F rows for one k-step: eight bytes per 64 rows
// (F a multiple of 4), a word for 32 rows, two bytes for 16. Byte 2 * (f % 2) +
// h of word f / 2 is fragment f, half h.
template <int F>
struct Scales {
  static constexpr int kWords = F < 2 ? 1 : F / 2;
  static_assert(F == 1 || F == 2 || F % 4 == 0, "fragments");
  uint32_t w[kWords];
  // rsrc: the scale tiles of a panel (rows from a multiple of 64 on); row: the
  // first of the wave's rows in it. Past the panel reads as zero.
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rsrc, int row, int col_tiles, int kt, int lane) {
    if (F >= 4) {
#pragma unroll
      for (int t = 0; t < F / 4; ++t) {
        const v2u v = __builtin_amdgcn_raw_buffer_load_b64(
            rsrc, (uint32_t)(((row >> 6) + t) * col_tiles) * 512 + lane * 8, kt * 512, 0);
        w[2 * t] = v.x;
        w[2 * t + 1] = v.y;
      }
    } else if (F == 2) {
      w[0] = __builtin_amdgcn_raw_buffer_load_b32(
          rsrc, (uint32_t)((row >> 6) * col_tiles) * 512 + lane * 8 + ((row >> 4) & 2) * 2, kt * 512, 0);
    } else {
      w[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(
          rsrc, (uint32_t)((row >> 6) * col_tiles) * 512 + lane * 8 + ((row >> 4) & 3) * 2, kt * 512, 0);
    }
  }
};

// ---------------------------------------------------------- tile kernel ----
// BM x BN outputs per workgroup, a wave (BM / WAVES_M) x (BN / WAVES_N) of them.
// Ring of S k-steps in LDS (1 KB blocks of 8 rows x 128 bytes, 16-byte chunk c of
// row R in slot c ^ (R % 8)). k-step kt: wait for its DMAs, barrier (which also
// says that every wave is done with k-step kt - 1), refill that slot with k-step
// kt + S - 1, multiply.
template <int BM, int BN, int WAVES_M, int WAVES_N, int S, int EPI>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N) void fp4_tile(Fp4Args p) {
  constexpr int BK = 128, NWAVES = WAVES_M * WAVES_N;
  constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, FM = WM / 16, FN = WN / 16;
  constexpr int A_BYTES = BM * BK, SLOT = (BM + BN) * BK;
  constexpr int BLOCKS = (BM + BN) / 8, LOADS = BLOCKS / NWAVES;
  static_assert(BM % 64 == 0 && BN % 64 == 0 && BLOCKS % NWAVES == 0 && S >= 2, "tile shape");
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
  const __amdgpu_buffer_rsrc_t rsa = row_rsrc(p.as + (m0 >> 6) * KT * 512, ((rows_a + 63) >> 6) * KT * 512);
  const __amdgpu_buffer_rsrc_t rsb = row_rsrc(p.bs + (n0 >> 6) * KT * 512, ((rows_b + 63) >> 6) * KT * 512);

  const int drow = lane >> 3;
  const int dchunk = ((lane & 7) ^ drow) * 16;
  // Past the last column of a row the lane asks for an offset past the buffer.
  auto issue = [&](int kt) {
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
  };
  const int r16 = lane & 15;
  const int rd_row = (r16 >> 3) * 1024 + (r16 & 7) * 128;
  auto frag = [&](const char* base, int f, int h) -> v4i {
    return *reinterpret_cast<const v4i*>(base + f * 2048 + rd_row + (((lane >> 4) + 4 * h) ^ (r16 & 7)) * 16);
  };

  v4f acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  Scales<FM> sa, sa_next;
  Scales<FN> sb, sb_next;
  sa.load(rsa, wm * WM, KT, 0, lane);
  sb.load(rsb, wn * WN, KT, 0, lane);
#pragma unroll
  for (int t = 0; t < S - 1; ++t) issue(t);
  constexpr int kVm = (S - 2) * LOADS;
  static_assert(kVm <= 63, "vmcnt range");
  constexpr int kWait = 0x70 | 0xf00 | (kVm & 0xf) | ((kVm >> 4) << 14);  // vmcnt(kVm)
#pragma unroll 1
  for (int kt = 0; kt < KT; ++kt) {
    // In flight: the DMAs of k-steps kt .. kt + S - 2, oldest first.
    __builtin_amdgcn_s_waitcnt(kWait);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    const int next = kt + 1 < KT ? kt + 1 : kt;
    sa_next.load(rsa, wm * WM, KT, next, lane);
    sb_next.load(rsb, wn * WN, KT, next, lane);
    __builtin_amdgcn_sched_barrier(0);  // the scale loads stay older than the DMAs (kWait counts those)
    issue(kt + S - 1);
    __builtin_amdgcn_sched_barrier(0);
    const char* const slot = smem + (kt % S) * SLOT;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v4i a[FM], w[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) w[j] = frag(slot + A_BYTES, wn * FN + j, h);
#pragma unroll
      for (int i = 0; i < FM; ++i) a[i] = frag(slot, wm * FM + i, h);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = mfma_fp4(w[j], a[i], acc[i][j], 2 * (j & 1) + h, sb.w[j >> 1], 2 * (i & 1) + h, sa.w[i >> 1]);
    }
    sa = sa_next;
    sb = sb_next;
  }
  __builtin_amdgcn_s_waitcnt(0x70 | 0xf00);  // vmcnt(0): the trailing DMAs have landed
  __syncthreads();
  if (p.staged) store_staged<FM, FN, EPI>(p, acc, smem + wave * STAGE, m0 + wm * WM, n0 + wn * WN, lane);
  else store_direct<FM, FN, EPI>(p, acc, m0 + wm * WM, n0 + wn * WN, lane);
}

template <int BM, int BN, int WAVES_M, int WAVES_N, int S>
int launch_tile(Fp4Args p, int epilogue, hipStream_t s) {
  const int64_t tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
  LR_REQUIRE(tm * tn <= kMaxBlocks, "mxfp4_gemm: %lld output tiles are not supported", (long long)(tm * tn));
  p.tiles_m = (int)tm;
  p.tiles_n = (int)tn;
  p.group_m = 8;
  const dim3 grid((unsigned)(tm * tn)), block(64 * WAVES_M * WAVES_N);
  if (epilogue == EPI_BF16) fp4_tile<BM, BN, WAVES_M, WAVES_N, S, EPI_BF16><<<grid, block, 0, s>>>(p);
  else if (epilogue == EPI_GELU) fp4_tile<BM, BN, WAVES_M, WAVES_N, S, EPI_GELU><<<grid, block, 0, s>>>(p);
  else fp4_tile<BM, BN, WAVES_M, WAVES_N, S, EPI_GATED><<<grid, block, 0, s>>>(p);
  return check_launch("mxfp4_gemm");
}

}  // namespace
}  // namespace lr

using namespace lr;

extern "C" int lr_mxfp4_gemm(const void* a, const void* a_scale, const void* b, const void* b_scale, int64_t m,
                             int64_t n, int64_t k, const void* bias, void* out, int epilogue, const void* residual,
                             const void* table, int64_t table_rows, int64_t table_width, const int64_t* indices,
                             int64_t sequence, int gate_slot, void* stream) {
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
  Fp4Args p = {};
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
  return launch_tile<128, 128, 2, 2, 2>(p, epilogue, as_stream(stream));
}
