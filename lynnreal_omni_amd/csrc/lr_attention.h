// lr_attention.h - one pass over a run of key tiles, shared by the attention kernels
// (attention.hip has the mathematics): operand layouts, the running maximum, and the
// loop over the tiles.
#pragma once

#include <math.h>

#include <type_traits>

#include "lr_device.h"

namespace lr {
namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

template <typename T> struct Mfma;
template <> struct Mfma<__bf16> {
  typedef v8bf V;
  static constexpr float kShift = 0.0f;
  static __device__ __forceinline__ v16f mul(const V& a, const V& b, const v16f& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf2(a, b); }
  static __device__ __forceinline__ float first(uint32_t w) { return bf_lo(w); }
  static __device__ __forceinline__ float second(uint32_t w) { return bf_hi(w); }
  static __device__ __forceinline__ float add2(uint32_t w, float l) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, w), __builtin_bit_cast(v2bf, 0x3f803f80u), l, false);
  }
};
template <> struct Mfma<_Float16> {
  typedef v8h V;
  // p is kept 2^7 larger: its subnormals then begin at 2^-31 of a row's largest.
  static constexpr float kShift = 7.0f;
  static __device__ __forceinline__ v16f mul(const V& a, const V& b, const v16f& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const v2h h = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, h);
  }
  static __device__ __forceinline__ float first(uint32_t w) { return (float)__builtin_bit_cast(v2h, w)[0]; }
  static __device__ __forceinline__ float second(uint32_t w) { return (float)__builtin_bit_cast(v2h, w)[1]; }
  static __device__ __forceinline__ float add2(uint32_t w, float l) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, w), __builtin_bit_cast(v2h, 0x3c003c00u), l, false);
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

template <typename V8>
__device__ __forceinline__ V8 tr_pair(const char* a0, const char* a1) {
  const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t)a0);
  const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t)a1);
  return __builtin_bit_cast(V8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}

constexpr int kRows = 128;       // rows per workgroup
constexpr int kKeys = 64;        // keys per tile
constexpr float kSlack = 8.0f;   // log2

// Sum of v over the lanes up to this one: within rows of 16 lanes by shifts, then the
// last lane of each row (and of each pair of rows) added to the rows behind it.
__device__ __forceinline__ int wave_prefix_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// Moves m to the new maximum x where some row of the wave exceeds it by more than
// the slack (or has its first key); returns what the exponent subtracts.
template <int DB, bool EXACT>
__device__ __forceinline__ float move_max(float x, float& m, float& l, float& exact, v16f (&o)[DB], float c, float shift) {
  if (__any((x - m) * c > kSlack || (m == -INFINITY && x > -INFINITY))) {
    const float mn = fmaxf(m, x);
    const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * c);
    m = mn;
    l *= alpha;
    if constexpr (EXACT) exact *= alpha;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
  }
  return m == -INFINITY ? 0.0f : m * c - shift;
}

// The keys and values of one cache, as `attend` reads them: tile t is keys 64 t .. of it.
struct OneCache {
  const uint16_t *k, *v;   // first key and value of the head
  int64_t kt, vt;          // strides between keys and between values
  int kn, sure, seen;      // keys; those that every row of the workgroup sees; those of the lane's row
  __device__ __forceinline__ int64_t stride(int, int is_v) const { return is_v ? vt : kt; }
  __device__ __forceinline__ const uint16_t* at(int t, int is_v) const {
    return (is_v ? v : k) + (int64_t)t * kKeys * stride(t, is_v);
  }
  __device__ __forceinline__ int left(int t) const { return kn - t * kKeys; }          // keys from tile t on
  __device__ __forceinline__ bool whole(int t) const { return (t + 1) * kKeys <= sure; }
  __device__ __forceinline__ int first(int t) const { return t * kKeys; }   // key of tile t
  __device__ __forceinline__ int limit(int) const { return seen; }          // keys that the row sees, counted as first() does
  static constexpr bool kOneStride = true;   // whether all tiles have the strides of the first
};

template <int D>
constexpr int kTileBytes = 2 * 2 * kKeys * 2 * D;   // LDS of a workgroup: two slots of K and V

// Four waves of 32 rows; keys in tiles of 64 through two slots of LDS (K rows,
// then V rows), by 16-byte DMA. A row's 16-byte chunk c lies in slot c ^ 2 * (row
// / (256 / row bytes) % (row bytes / 32)): eight rows' equal 32-byte columns are
// on distinct banks, which is what both reads need.
//
// A trip computes the scores of tile t + 1 while those of tile t become
// probabilities, then the second product of tile t while the maxima of tile t + 1
// form: the matrix instructions of each phase are independent of its vector work.
// The compiler would move the exponentials behind the first product (the fences
// and the empty asm keep them between its instructions). Two workgroups share a
// CU (256 registers, 64 KB), so that one wave's vector phase runs under the
// other's matrix phase; the second product's priority is raised.
// Measured, 56 heads of 128, 12605 tokens, bf16: without the pipeline and with one
// wave per SIMD 6.5 ms; two waves per SIMD 4.42; pipelined 4.25; two tiles per
// trip (no copies of the scores, constant LDS slots) and the priority 4.10-4.14
// ms, 1100-1110 TFLOP/s. There the clock is down to 1.69 GHz and the matrix units
// are 62% busy: the chip's power is the bound, as for a large bf16 matrix product
// (1505 TFLOP/s on the same card). 64 rows per wave and one wave per SIMD halves
// the LDS reads and was slower (869 against 734 us on 8 heads), reading V by asm
// blocks with their waits too (4.32 ms).
// FEW, a wave's rows: what counts is the stream of keys, 32 KB in flight per workgroup;
// waves without rows only load. No pipeline: the next tile is in flight while this one
// is worked on, and the second product runs twice, for p rounded and for what the
// rounding left, so that the output's rounding is all that remains (error against 64
// bits 1.35 times smaller for long caches; 1 to 4% of the time, 4 to 13% with 64 to 128
// rows, which do without). One token of 56 heads over 131072 keys of 8 (537 MB): 107-109
// us with the join of 64 splits, 5.0 TB/s, as fast as a copy. Keys straight into
// registers by waves that share nothing and meet no barrier: 129 us.
//
// Adds tiles t0 .. t1 - 1 to the row's m, l and o (from -inf, 0 and 0). A lane holds columns
// 32 * d + 8 * g + 4 * half + 0..3 of row `col` of its wave; l and the exact sum are over
// its own keys, the partner lane l ^ 32 has the others. EXACT: the sum of the unrounded
// weights too, which the logarithm of the row's sum needs (l is that where FEW).
// `smem`: kTileBytes<D> bytes; every thread of the workgroup takes part.
template <typename T, int D, bool FEW, bool EXACT, class Keys>
__device__ __forceinline__ void attend(char* smem, const Keys& keys, const uint16_t* qrow, const float c, const int t0,
                                       const int t1, const bool idle, float& m, float& l, float& exact, float& off,
                                       v16f (&o)[D / 32]) {
  typedef typename Mfma<T>::V V8;
  constexpr int WAVES = kRows / 32;
  constexpr int ROW = 2 * D;                     // bytes of a row
  constexpr int CH = ROW / 16;                   // chunks per row
  constexpr int RPB = 256 / ROW, PAIRS = ROW / 32;
  constexpr int TILE = kKeys * ROW, SLOT = 2 * TILE;
  constexpr int DMAS = TILE / 1024 / WAVES;      // per wave, operand and tile
  constexpr int KD = D / 16, DB = D / 32;
  static_assert(TILE / 1024 % WAVES == 0, "DMA split");
  static_assert(2 * SLOT == kTileBytes<D>, "LDS");
  constexpr float kShift = Mfma<T>::kShift;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int half = lane >> 5, col = lane & 31;
  V8 q[KD];
#pragma unroll
  for (int d = 0; d < KD; ++d) q[d] = *reinterpret_cast<const V8*>(qrow + 16 * d + 8 * half);

  // DMA i of this wave: 1 KB of the tile's rows.
  uint32_t koff[DMAS], voff[DMAS];
  auto offset = [&](int i, uint32_t stride) __attribute__((always_inline)) {
    const int at = (wave * DMAS + i) * 64 + lane;  // 16-byte slot of the tile
    const int row = at / CH, ch = at % CH ^ (row / RPB % PAIRS) * 2;
    return (uint32_t)row * stride * 2 + ch * 16;
  };
  if constexpr (Keys::kOneStride) {
#pragma unroll
    for (int i = 0; i < DMAS; ++i) {
      koff[i] = offset(i, (uint32_t)keys.stride(t0, 0));
      voff[i] = offset(i, (uint32_t)keys.stride(t0, 1));
    }
  }
  auto issue = [&](int t, int v) {
    if (t >= t1) return;
    char* const slot = smem + ((t - t0) & 1) * SLOT + v * TILE;
    const int left = min(kKeys, keys.left(t));  // rows past the last key read as zero
    const int64_t stride = keys.stride(t, v);
    const __amdgpu_buffer_rsrc_t r = row_rsrc(keys.at(t, v), ((int64_t)(left - 1) * stride + D) * 2);
#pragma unroll
    for (int i = 0; i < DMAS; ++i)
      dma16(r, slot + (wave * DMAS + i) * 1024,
            Keys::kOneStride ? (v ? voff[i] : koff[i]) : offset(i, (uint32_t)stride));
  };

  v16f s0[2], s1[2];
  float mx;
  uint32_t pk[4][4];
  m = -INFINITY;
  l = exact = off = 0.0f;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
  // Fragment reads. K: d = g / 2, rows 32 * (g % 2) + col, columns 16 * d + 8 *
  // half. V^T: 16 keys kc = g / DB, column 32 * (g % DB) + col, keys 16 * kc + 4 *
  // half + (0..3, 8..11).
  const int krow = col * ROW, kswz = (col / RPB % PAIRS) * 2;
  auto kfrag = [&](const char* ks, int g) -> V8 {
    return *reinterpret_cast<const V8*>(ks + (g & 1) * 32 * ROW + krow + ((2 * (g >> 1) + half) ^ kswz) * 16);
  };
  const int i16 = lane & 15;
  const int vr = 4 * half + (i16 >> 2);
  auto vfrag = [&](const char* vs, int g) -> V8 {
    const int kc = g / DB, d = g % DB;
    const int c = 4 * d + 2 * ((lane >> 4) & 1) + (i16 >> 1 & 1);
    const int sub = (i16 & 1) * 8;
    return tr_pair<V8>(vs + (16 * kc + vr) * ROW + (c ^ (vr / RPB % PAIRS) * 2) * 16 + sub,
                       vs + (16 * kc + 8 + vr) * ROW + (c ^ ((vr + 8) / RPB % PAIRS) * 2) * 16 + sub);
  };
  constexpr int NQ = 2 * KD, NV = 4 * DB;   // matrix instructions of the two products
  constexpr int NP = 16, NP1 = 12;          // pairs of keys per lane; those under the first product
  auto pair = [&](v16f (&sc)[2], int j) {
    const int kc = j >> 2, w = j & 3, e = (kc & 1) * 8 + 2 * w;
    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kc >> 1][e], c, -off));
    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kc >> 1][e + 1], c, -off));
    pk[kc][w] = Mfma<T>::pack(p0, p1);
    l = Mfma<T>::add2(pk[kc][w], l);
    if constexpr (EXACT) exact += p0 + p1;
    asm volatile("" : "+v"(pk[kc][w]), "+v"(l));
  };
  auto masked = [&](v16f (&nx)[2], int t) {
    if (keys.whole(t)) return;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = keys.first(t) + 32 * kb + 8 * (e >> 2) + 4 * half + (e & 3);
        nx[kb][e] = key < keys.limit(t) ? nx[kb][e] : -INFINITY;
      }
  };
  auto score = [&](v16f (&nx)[2], const V8& kf, int g) {
    if (g < 2) {
#pragma unroll
      for (int e = 0; e < 16; ++e) nx[g][e] = 0.0f;
    }
    nx[g & 1] = Mfma<T>::mul(kf, q[g >> 1], nx[g & 1]);
  };
  // Publishes what every wave's DMAs have fetched, and frees the slots that they
  // go to next: behind it every wave is done with tile t - 1.
  auto publish = [&]() {
    __builtin_amdgcn_s_waitcnt(0x70 | 0xf00);  // vmcnt(0)
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // Tile t, in slot `par`, with the scores sc; those of tile t + 1 go to nx.
  auto body = [&](v16f (&sc)[2], v16f (&nx)[2], int t, const int par, auto has_next) {
    constexpr bool NEXT = decltype(has_next)::value;
    const char* const ks = smem + (par ^ 1) * SLOT;
    const char* const vs = smem + par * SLOT + TILE;
    V8 kf[4], vf[4];
    __builtin_amdgcn_s_setprio(0);
    if constexpr (NEXT) {
#pragma unroll
      for (int g = 0; g < 3; ++g) kf[g] = kfrag(ks, g);
#pragma unroll
      for (int g = 0; g < NQ; ++g) {
        if (g + 3 < NQ) kf[(g + 3) & 3] = kfrag(ks, g + 3);
        else vf[(g + 3 - NQ) & 3] = vfrag(vs, g + 3 - NQ);
        score(nx, kf[g & 3], g);
#pragma unroll
        for (int j = 0; j < NP1; ++j)
          if (j * NQ / NP1 == g) pair(sc, j);
        __builtin_amdgcn_sched_barrier(0);
      }
      masked(nx, t + 1);
      mx = -INFINITY;
    } else {
#pragma unroll
      for (int g = 0; g < 3; ++g) vf[g] = vfrag(vs, g);
#pragma unroll
      for (int j = 0; j < NP1; ++j) pair(sc, j);
    }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int g = 0; g < NV; ++g) {
      const int kc = g / DB;
      if (g + 3 < NV) vf[(g + 3) & 3] = vfrag(vs, g + 3);
      const uint4 pw = make_uint4(pk[kc][0], pk[kc][1], pk[kc][2], pk[kc][3]);
      o[g % DB] = Mfma<T>::mul(vf[g & 3], __builtin_bit_cast(V8, pw), o[g % DB]);
#pragma unroll
      for (int j = NP1; j < NP; ++j)
        if ((j - NP1) * (NV / 2) / (NP - NP1) == g) pair(sc, j);
      if constexpr (NEXT) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (j * NV / 16 == g) mx = fmaxf(fmaxf(mx, nx[j >> 3][2 * j & 15]), nx[j >> 3][(2 * j & 15) + 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto advance = [&]() { off = move_max<DB, EXACT && !FEW>(max_with_partner(mx), m, l, exact, o, c, kShift); };

  if constexpr (FEW) {
    uint32_t lo[4][4];
    if (t0 < t1) {
      issue(t0, 0);
      issue(t0, 1);
    }
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      publish();
      issue(t + 1, 0);
      issue(t + 1, 1);
      if (idle) continue;   // without rows: loads and barriers alone
      const char* const ks = smem + ((t - t0) & 1) * SLOT;
      const char* const vs = ks + TILE;
#pragma unroll
      for (int g = 0; g < NQ; ++g) score(s0, kfrag(ks, g), g);
      masked(s0, t);
      mx = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s0[kb][e]);
      advance();
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int kc = j >> 2, w = j & 3, e = (kc & 1) * 8 + 2 * w;
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s0[kc >> 1][e], c, -off));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s0[kc >> 1][e + 1], c, -off));
        pk[kc][w] = Mfma<T>::pack(p0, p1);
        lo[kc][w] = Mfma<T>::pack(p0 - Mfma<T>::first(pk[kc][w]), p1 - Mfma<T>::second(pk[kc][w]));
        l += p0 + p1;
      }
#pragma unroll
      for (int g = 0; g < NV; ++g) {
        const int kc = g / DB;
        const V8 vf = vfrag(vs, g);
        const uint4 hi4 = make_uint4(pk[kc][0], pk[kc][1], pk[kc][2], pk[kc][3]);
        const uint4 lo4 = make_uint4(lo[kc][0], lo[kc][1], lo[kc][2], lo[kc][3]);
        o[g % DB] = Mfma<T>::mul(vf, __builtin_bit_cast(V8, hi4), o[g % DB]);
        o[g % DB] = Mfma<T>::mul(vf, __builtin_bit_cast(V8, lo4), o[g % DB]);
      }
    }
  } else if (t0 < t1 && idle) {
    // A wave without rows takes part in the loads and barriers alone.
    issue(t0, 0);
    publish();
    issue(t0 + 1, 0);
    issue(t0, 1);
#pragma unroll 1
    for (int t = t0; t + 1 < t1; ++t) {
      publish();
      issue(t + 2, 0);
      issue(t + 1, 1);
    }
    publish();
  } else if (t0 < t1) {
    // K(t + 1) and V(t) are used together; K(t0) alone first.
    issue(t0, 0);
    publish();
    issue(t0 + 1, 0);
    issue(t0, 1);
#pragma unroll
    for (int g = 0; g < NQ; ++g) score(s0, kfrag(smem, g), g);
    masked(s0, t0);
    mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s0[kb][e]);
    auto step = [&](v16f (&sc)[2], v16f (&nx)[2], int t, const int par) {
      advance();
      publish();
      issue(t + 2, 0);
      issue(t + 1, 1);
      body(sc, nx, t, par, std::true_type{});
    };
    int t = t0;
#pragma unroll 1
    for (; t + 2 < t1; t += 2) {
      step(s0, s1, t, 0);
      step(s1, s0, t + 1, 1);
    }
    if (t + 1 < t1) {
      step(s0, s1, t, 0);
      advance();
      publish();
      body(s1, s0, t1 - 1, 1, std::false_type{});
    } else {
      advance();
      publish();
      body(s0, s1, t1 - 1, 0, std::false_type{});
    }
  }
  if constexpr (FEW) exact = l;
}

}  // namespace
}  // namespace lr
