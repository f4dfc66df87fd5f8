// lr_mxfp4_rows.h - eight values of a row as loaded, their largest magnitude and
// their E2M1 codes, for the kernels that quantize rows (mxfp4.hip gives the format).
#pragma once

#include "lr_device.h"
#include "lr_runtime.h"

namespace lr {
namespace {

typedef unsigned short v2us __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

// Eight values of a row as loaded, the bits of their largest magnitude as
// fp32, and their codes.
template <int DTYPE>
struct Row8;

// Largest of the 2 x 4 magnitudes of 16-bit floats, as 16 bits: magnitudes
// order like integers, with a NaN above the infinities.
__device__ __forceinline__ uint32_t magnitude16(const uint4& v) {
  auto two = [](uint32_t w) { return __builtin_bit_cast(v2us, w & 0x7fff7fffu); };
  v2us m = __builtin_elementwise_max(__builtin_elementwise_max(two(v.x), two(v.y)),
                                     __builtin_elementwise_max(two(v.z), two(v.w)));
  return m[0] > m[1] ? m[0] : m[1];
}

template <>
struct Row8<LR_DTYPE_BF16> {
  static constexpr int kBytes = 2;
  uint4 v;
  __device__ void load(const char* p) { v = load_nt(reinterpret_cast<const uint4*>(p)); }
  __device__ void load(__amdgpu_buffer_rsrc_t r, uint32_t offset) { v = buf_load16(r, offset); }
  __device__ void load_some(const char* p, int n) {
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = i < n ? reinterpret_cast<const uint16_t*>(p)[i] : 0u;
    v = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
  }
  __device__ uint32_t magnitude() const { return magnitude16(v) << 16; }
  __device__ uint32_t codes(float scale) const {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(v2bf, v.x), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(v2bf, v.y), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(v2bf, v.z), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(v2bf, v.w), scale, 3);
  }
};

template <>
struct Row8<LR_DTYPE_F16> {
  static constexpr int kBytes = 2;
  uint4 v;
  __device__ void load(const char* p) { v = load_nt(reinterpret_cast<const uint4*>(p)); }
  __device__ void load(__amdgpu_buffer_rsrc_t r, uint32_t offset) { v = buf_load16(r, offset); }
  __device__ void load_some(const char* p, int n) {
    Row8<LR_DTYPE_BF16> r;
    r.load_some(p, n);
    v = r.v;
  }
  __device__ uint32_t magnitude() const {
    return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)magnitude16(v)));
  }
  __device__ uint32_t codes(float scale) const {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(v2h, v.x), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(v2h, v.y), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(v2h, v.z), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(v2h, v.w), scale, 3);
  }
};

template <>
struct Row8<LR_DTYPE_F32> {
  static constexpr int kBytes = 4;
  uint32_t w[8];
  __device__ void load(const char* p) {
    const uint4 a = load_nt(reinterpret_cast<const uint4*>(p));
    const uint4 b = load_nt(reinterpret_cast<const uint4*>(p) + 1);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  }
  __device__ void load(__amdgpu_buffer_rsrc_t r, uint32_t offset) {
    const uint4 a = buf_load16(r, offset), b = buf_load16(r, offset + 16);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  }
  __device__ void load_some(const char* p, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = i < n ? reinterpret_cast<const uint32_t*>(p)[i] : 0u;
  }
  __device__ uint32_t magnitude() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m;
  }
  __device__ uint32_t codes(float scale) const {
    auto f = [&](int i) { return __uint_as_float(w[i]); };
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f(0), f(1), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f(2), f(3), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f(4), f(5), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f(6), f(7), scale, 3);
  }
};

// Lane l takes the larger of its value and lane l ^ 1's, then l ^ 2's: the
// largest of the quad that holds a block.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));
}

// E8M0 byte of a block from the fp32 bits of its largest magnitude.
__device__ __forceinline__ uint32_t scale_byte(uint32_t magnitude) {
  const int field = (int)(magnitude >> 23);
  return field == 255 ? 255u : (uint32_t)max(field - 2, 0);
}

}  // namespace
}  // namespace lr
