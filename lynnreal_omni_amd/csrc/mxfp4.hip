// mxfp4.hip - rows to microscaled 4-bit floating point (MXFP4) and back.
//
// A row is cut into blocks of 32 (the last one filled up with zeros). A block
// with largest magnitude a is 2^e times 32 values of 0, 0.5, 1, 1.5, 2, 3, 4, 6
// with a sign (E2M1):
//   e    = max(floor(log2(a)) - 2, -127)   so that a / 2^e lies in [4, 8)
//   code = the E2M1 value nearest to x / 2^e, ties to the even code, past 6 : 6
// x / 2^e is exact, so the only rounding is the one to the code. e is kept as
// e + 127 in a byte (E8M0), the fp32 exponent field of a less 2. A block with a
// NaN or an infinity gets the byte 255, which stands for NaN here and in the
// matrix instruction: products of its row are NaN, never a finite wrong value.
//
// Codes: two per byte, the even column in the low half; ceil(width / 32) * 16
// bytes per row. Scales lie as the matrix instruction takes them (lr_mxfp4.h):
// 512 bytes for 64 rows x 8 blocks, so both kernels work on tiles of 256
// columns, and one tile's scales are written as whole cache lines.
#include "lr_device.h"
#include "lr_mxfp4.h"
#include "lr_mxfp4_rows.h"
#include "lr_runtime.h"

namespace lr {
namespace {

// One workgroup quantizes GROUPS * 16 rows x 256 columns. A wave reads two rows
// per step, eight values (a quarter of a block) per lane: 512 contiguous bytes
// of a row in, 128 out. Four lanes agree on a block's magnitude without LDS;
// the scale bytes of the tile meet in LDS and leave as whole words. Bound by HBM:
// 12605 x 14336 bf16 in 70-75 us, 6.1-6.5 TB/s (four bytes read for one written);
// 878 x 5376 in 3.8 us, 1 row in 2.4.
template <int DTYPE, int GROUPS, bool VECTOR>
__global__ __launch_bounds__(256) void quantize_mxfp4(const char* __restrict__ x, int64_t rows, int64_t width,
                                                      uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                      int col_tiles) {
  constexpr int kRows = 16 * GROUPS, kSteps = kRows / 8;
  typedef Row8<DTYPE> R;
  // Scale byte of (row 16 * f + r, block 4 * h + g) at [16 * g + r][2 * f + h].
  __shared__ __attribute__((aligned(16))) uint8_t tile[64][2 * GROUPS];
  const int64_t row0 = (int64_t)(blockIdx.x / col_tiles) * kRows;
  const int ct = (int)(blockIdx.x % col_tiles);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t blocks = (width + 31) >> 5;
  const int chunk = lane & 31;                      // eight columns of the tile's 256
  const int64_t col = (int64_t)ct * 256 + chunk * 8;
  const int block = chunk >> 2;
  const bool column = (int64_t)ct * 8 + block < blocks;
  R v[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int64_t row = row0 + s * 8 + wave * 2 + (lane >> 5);
    const char* p = x + (row * width + col) * R::kBytes;
    if (VECTOR) {
      // width % 8 == 0: a chunk lies in the row or past it as a whole.
      if (row < rows && col < width) v[s].load(p);
      else v[s] = R{};
    } else {
      const int64_t left = row < rows ? width - col : 0;
      v[s].load_some(p, left >= 8 ? 8 : (left > 0 ? (int)left : 0));
    }
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int r = s * 8 + wave * 2 + (lane >> 5);
    const int64_t row = row0 + r;
    const uint32_t byte = scale_byte(quad_max(v[s].magnitude()));
    if ((lane & 3) == 0) tile[16 * (block & 3) + (r & 15)][2 * (r >> 4) + (block >> 2)] = (uint8_t)byte;
    if (row >= rows || !column) continue;
    // 2^e as fp32 is the byte in the exponent field; e = -127 is a subnormal.
    const float scale = __uint_as_float(byte == 0 ? 0x00400000u : byte << 23);
    const uint32_t c = byte == 255 ? 0u : v[s].codes(scale);
    *reinterpret_cast<uint32_t*>(codes + (row * blocks + ct * 8) * 16 + chunk * 4) = c;
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    // GROUPS * 2 bytes of each lane's 8; 16-row groups of one tile go to several workgroups.
    uint8_t* dst = scales + ((row0 >> 6) * col_tiles + ct) * 512 + threadIdx.x * 8 + 2 * ((row0 >> 4) & 3);
    if (GROUPS == 4)
      *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(tile[threadIdx.x]);
    else
      *reinterpret_cast<uint16_t*>(dst) = *reinterpret_cast<const uint16_t*>(tile[threadIdx.x]);
  }
}

template <int DTYPE>
__device__ __forceinline__ void store8(void* out, int64_t at, const float f[8], int n) {
  if (DTYPE == LR_DTYPE_F32) {
    float* o = static_cast<float*>(out) + at;
    if (n == 8 && at % 4 == 0) {
      reinterpret_cast<float4*>(o)[0] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(o)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) o[i] = f[i];
    }
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (DTYPE == LR_DTYPE_BF16) {
      w[i] = pack_bf2(f[2 * i], f[2 * i + 1]);
    } else {
      const v2h h = {(_Float16)f[2 * i], (_Float16)f[2 * i + 1]};
      w[i] = __builtin_bit_cast(uint32_t, h);
    }
  }
  uint16_t* o = static_cast<uint16_t*>(out) + at;
  if (n == 8 && at % 8 == 0) {
    store_nt(reinterpret_cast<uint4*>(o), make_uint4(w[0], w[1], w[2], w[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) o[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
  }
}

// The inverse: 16 rows x 256 columns per workgroup, eight codes (one word) per
// lane and step. A code's magnitude is a 16-entry table in two registers'
// bytes: twice the value, 0 1 2 3 4 6 8 12, picked by v_perm; the scale is then
// one power of two lower. Exact in bf16 and fp32; fp16 rounds and overflows as
// a conversion from fp32 does. Bound by its stores: 12605 x 14336 to bf16 in 70-85
// us, 5.4-6.5 TB/s.
template <int DTYPE>
__global__ __launch_bounds__(256) void dequantize_mxfp4(const uint8_t* __restrict__ codes,
                                                        const uint8_t* __restrict__ scales, int64_t rows,
                                                        int64_t width, void* __restrict__ out, int col_tiles) {
  const int64_t row0 = (int64_t)(blockIdx.x / col_tiles) * 16;
  const int ct = (int)(blockIdx.x % col_tiles);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t blocks = (width + 31) >> 5;
  const int chunk = lane & 31, block = chunk >> 2;
  const int64_t col = (int64_t)ct * 256 + chunk * 8;
  if (col >= width) return;
  uint32_t c[2], e[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int64_t row = row0 + s * 8 + wave * 2 + (lane >> 5);
    const int64_t at = row < rows ? row : rows - 1;
    c[s] = *reinterpret_cast<const uint32_t*>(codes + (at * blocks + ct * 8) * 16 + chunk * 4);
    e[s] = scales[mxfp4_scale_at(at, (int64_t)ct * 8 + block, col_tiles)];
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int64_t row = row0 + s * 8 + wave * 2 + (lane >> 5);
    if (row >= rows) continue;
    // Half of 2^(e - 127); 255 stands for NaN.
    const float half = e[s] == 255 ? __uint_as_float(0x7fc00000u)
                                   : __uint_as_float(e[s] > 1 ? (e[s] - 1) << 23 : 0x00200000u << e[s]);
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t code = c[s] >> (4 * i);
      const uint32_t twice = __builtin_amdgcn_perm(0x0c080604u, 0x03020100u, (code & 7u) | 0x0c0c0c00u) & 0xffu;
      f[i] = __uint_as_float(__float_as_uint((float)twice) | (code & 8u) << 28) * half;
    }
    const int64_t left = width - col;
    store8<DTYPE>(out, row * width + col, f, left >= 8 ? 8 : (int)left);
  }
}

int check_rows(int64_t rows, int64_t width, const char* what) {
  LR_REQUIRE(rows >= 0 && width >= 0, "%s: negative shape [%lld, %lld]", what, (long long)rows, (long long)width);
  LR_REQUIRE(width <= (1LL << 30), "%s: %lld columns are not supported", what, (long long)width);
  return LR_OK;
}

}  // namespace

// Launches over at most kMaxBlocks workgroups, in slices of whole scale tiles.
template <class F>
static int by_slices(int64_t rows, int rows_per_block, int64_t col_tiles, F launch) {
  const int64_t tiles = kMaxBlocks / col_tiles * rows_per_block / 64;   // of 64 rows
  const int64_t step = (tiles < 1 ? 1 : tiles) * 64;
  for (int64_t first = 0; first < rows; first += step) {
    const int64_t n = rows - first < step ? rows - first : step;
    launch(first, n, (unsigned)((n + rows_per_block - 1) / rows_per_block * col_tiles));
    if (int rc = check_launch("mxfp4")) return rc;
  }
  return LR_OK;
}

template <int DTYPE>
static int quantize(const void* x, int64_t rows, int64_t width, void* codes, void* scales, hipStream_t s) {
  const int64_t col_tiles = mxfp4_scale_tiles(width);
  const bool vector = width % 8 == 0 && aligned(x, 16);
  // 64 rows per workgroup write their scales as whole lines; with few rows 16
  // spread over more CUs: 878 x 5376 (294 tiles) 3.6 us with 16 and 4.8 with 64, 2048 x
  // 5120 (640) 6.3 and 6.8, 3683 x 5376 (1218) 10.9 and 10.3, 12605 x 5376 31.9 and 29.1.
  const bool large = (rows + 63) / 64 * col_tiles >= 4 * compute_units();
  const int64_t blocks = (width + 31) / 32;
  return by_slices(rows, large ? 64 : 16, col_tiles, [&](int64_t first, int64_t n, unsigned grid) {
    const char* px = static_cast<const char*>(x) + first * width * Row8<DTYPE>::kBytes;
    uint8_t* pc = static_cast<uint8_t*>(codes) + first * blocks * 16;
    uint8_t* ps = static_cast<uint8_t*>(scales) + first / 64 * col_tiles * 512;
    if (large) {
      if (vector) quantize_mxfp4<DTYPE, 4, true><<<grid, 256, 0, s>>>(px, n, width, pc, ps, (int)col_tiles);
      else quantize_mxfp4<DTYPE, 4, false><<<grid, 256, 0, s>>>(px, n, width, pc, ps, (int)col_tiles);
    } else {
      if (vector) quantize_mxfp4<DTYPE, 1, true><<<grid, 256, 0, s>>>(px, n, width, pc, ps, (int)col_tiles);
      else quantize_mxfp4<DTYPE, 1, false><<<grid, 256, 0, s>>>(px, n, width, pc, ps, (int)col_tiles);
    }
  });
}

}  // namespace lr

using namespace lr;

extern "C" int lr_quantize_rows_mxfp4(const void* x, int dtype, int64_t rows, int64_t width, void* codes,
                                      void* scales, void* stream) {
  if (int rc = check_rows(rows, width, "quantize_rows_mxfp4")) return rc;
  LR_REQUIRE(dtype == LR_DTYPE_BF16 || dtype == LR_DTYPE_F16 || dtype == LR_DTYPE_F32,
             "quantize_rows_mxfp4: unknown dtype %d", dtype);
  if (rows == 0 || width == 0) return LR_OK;
  LR_REQUIRE(x && codes && scales, "quantize_rows_mxfp4: null pointer");
  LR_REQUIRE(aligned(x, dtype == LR_DTYPE_F32 ? 4 : 2) && aligned(codes, 16) && aligned(scales, 16),
             "quantize_rows_mxfp4: codes and scales must be 16-byte aligned");
  hipStream_t s = as_stream(stream);
  if (dtype == LR_DTYPE_BF16) return quantize<LR_DTYPE_BF16>(x, rows, width, codes, scales, s);
  if (dtype == LR_DTYPE_F16) return quantize<LR_DTYPE_F16>(x, rows, width, codes, scales, s);
  return quantize<LR_DTYPE_F32>(x, rows, width, codes, scales, s);
}

extern "C" int lr_dequantize_rows_mxfp4(const void* codes, const void* scales, int dtype, int64_t rows,
                                        int64_t width, void* out, void* stream) {
  if (int rc = check_rows(rows, width, "dequantize_rows_mxfp4")) return rc;
  LR_REQUIRE(dtype == LR_DTYPE_BF16 || dtype == LR_DTYPE_F16 || dtype == LR_DTYPE_F32,
             "dequantize_rows_mxfp4: unknown dtype %d", dtype);
  if (rows == 0 || width == 0) return LR_OK;
  LR_REQUIRE(codes && scales && out, "dequantize_rows_mxfp4: null pointer");
  LR_REQUIRE(aligned(codes, 16) && aligned(scales, 16) && aligned(out, 16),
             "dequantize_rows_mxfp4: pointers must be 16-byte aligned");
  const int64_t col_tiles = mxfp4_scale_tiles(width), blocks = (width + 31) / 32;
  hipStream_t s = as_stream(stream);
  return by_slices(rows, 16, col_tiles, [&](int64_t first, int64_t n, unsigned grid) {
    const uint8_t* pc = static_cast<const uint8_t*>(codes) + first * blocks * 16;
    const uint8_t* ps = static_cast<const uint8_t*>(scales) + first / 64 * col_tiles * 512;
    char* po = static_cast<char*>(out) + first * width * (dtype == LR_DTYPE_F32 ? 4 : 2);
    if (dtype == LR_DTYPE_BF16)
      dequantize_mxfp4<LR_DTYPE_BF16><<<grid, 256, 0, s>>>(pc, ps, n, width, po, (int)col_tiles);
    else if (dtype == LR_DTYPE_F16)
      dequantize_mxfp4<LR_DTYPE_F16><<<grid, 256, 0, s>>>(pc, ps, n, width, po, (int)col_tiles);
    else
      dequantize_mxfp4<LR_DTYPE_F32><<<grid, 256, 0, s>>>(pc, ps, n, width, po, (int)col_tiles);
  });
}
