// MXFP4 codec: 32 elements share one E8M0 scale, each is an e2m1 number.
//
//   e      = max(floor(log2 max|x|) - 2, -127)       (2: the exponent of 4)
//   scale  = e + 127                                 (255: NaN)
//   code_i = e2m1(x_i / 2^e), to nearest, ties to even, saturated at 6
//
// The scale is a power of two, so x / 2^e is exact and the code is the one
// rounding of the format.  A block that holds a NaN or an infinity has no
// scale: its byte is 255 and the whole block stands for NaN.
//
// Bound by memory: 2 (4) bytes read and 17/32 written an element.  Four lanes
// hold a block (16 bytes of bf16 each, so a wave reads 1 KiB in one go), the
// maximum is taken over the block's bit patterns (as integers: a NaN stays
// the largest) with two lane exchanges in the VALU, and the conversion
// instruction, which divides by the scale, makes two codes at a time.  16384 x
// 4096 bf16: 31-34 us, 5.0-5.5 TB/s (50 with the borders compared one by one);
// back again 28.5 us.
#include "common.hpp"
#include "experts.hpp"
#include "kernels.hpp"

namespace kiosk {
namespace {

constexpr int kThreads = 256;

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;

// Eight elements of a row; the exponent field of the largest among the four
// lanes of a block; eight codes.
struct Eight16 {
  uint32_t w[4];
  __device__ __forceinline__ explicit Eight16(const uint16_t* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
  __device__ __forceinline__ uint32_t peak() const {
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = __builtin_elementwise_max(
          m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
    return static_cast<uint32_t>(max(m[0], m[1])) << 16;
  }
  __device__ __forceinline__ uint32_t codes(float scale) const {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
        c, __builtin_bit_cast(bf16x2, w[0]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
        c, __builtin_bit_cast(bf16x2, w[1]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
        c, __builtin_bit_cast(bf16x2, w[2]), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
        c, __builtin_bit_cast(bf16x2, w[3]), scale, 3);
  }
};

struct Eight32 {
  float v[8];
  __device__ __forceinline__ explicit Eight32(const float* p) {
    const float4 lo = *reinterpret_cast<const float4*>(p);
    const float4 hi = *reinterpret_cast<const float4*>(p + 4);
    v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
    v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
  }
  __device__ __forceinline__ uint32_t peak() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ uint32_t codes(float scale) const {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
  }
};

// the larger of this lane's and its quad neighbour's (CTRL: which one)
template <int CTRL>
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  return max(v, static_cast<uint32_t>(
                    __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false)));
}

template <typename T, typename Eight>
__global__ __launch_bounds__(kThreads) void quantize_kernel(
    const T* __restrict__ x, uint32_t* __restrict__ codes,
    uint8_t* __restrict__ scales, size_t chunks) {
  const size_t stride = static_cast<size_t>(gridDim.x) * kThreads;
  // a block's four lanes are all inside or all outside (chunks % 4 == 0)
  for (size_t c = blockIdx.x * static_cast<size_t>(kThreads) + threadIdx.x;
       c < chunks; c += stride) {
    const Eight v(x + c * 8);
    const uint32_t peak = quad_max<0x4e>(quad_max<0xb1>(v.peak()));
    const int field = static_cast<int>(peak >> 23);
    const int byte = field == 255 ? 255 : max(field - 2, 0);
    // 2^(byte - 127): a number below the normal ones for byte 0
    const float scale =
        __uint_as_float(byte == 0 ? 0x00400000u : static_cast<uint32_t>(byte)
                                                      << 23);
    codes[c] = byte == 255 ? 0u : v.codes(scale);
    if ((c & 3) == 0) scales[c >> 2] = static_cast<uint8_t>(byte);
  }
}

__device__ __forceinline__ float value(uint32_t code, int byte) {
  // e2m1 magnitudes doubled: 0 1 2 3 4 6 8 12
  const uint32_t twice = (0xc8643210u >> (4 * (code & 7))) & 15u;
  const float v = ldexpf(static_cast<float>(twice), byte - 128);
  return byte == 255 ? __builtin_nanf("") : (code & 8) ? -v : v;
}

__device__ __forceinline__ void store8(uint16_t* p, const float (&v)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    u[i] = f32_to_bf16(v[2 * i]) |
           (static_cast<uint32_t>(f32_to_bf16(v[2 * i + 1])) << 16);
  *reinterpret_cast<uint4*>(p) = uint4{u[0], u[1], u[2], u[3]};
}

__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = float4{v[0], v[1], v[2], v[3]};
  *reinterpret_cast<float4*>(p + 4) = float4{v[4], v[5], v[6], v[7]};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(
    const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales,
    T* __restrict__ out, size_t chunks) {
  const size_t stride = static_cast<size_t>(gridDim.x) * kThreads;
  for (size_t c = blockIdx.x * static_cast<size_t>(kThreads) + threadIdx.x;
       c < chunks; c += stride) {
    const uint32_t word = codes[c];
    const int byte = scales[c >> 2];
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = value((word >> (4 * i)) & 15u, byte);
    store8(out + c * 8, v);
  }
}

unsigned grid_for(size_t chunks) {
  const size_t blocks = (chunks + kThreads - 1) / kThreads;
  return static_cast<unsigned>(blocks < 65536 ? blocks : 65536);
}

}  // namespace

hipError_t launch_mxfp4_quantize(const void* x, int bf16, uint8_t* codes,
                                 uint8_t* scales, size_t n,
                                 hipStream_t stream) {
  if (n % 32 != 0) return hipErrorInvalidValue;
  if (n == 0) return hipSuccess;
  const size_t chunks = n / 8;
  auto* words = reinterpret_cast<uint32_t*>(codes);
  const dim3 grid(grid_for(chunks)), block(kThreads);
  return bf16 ? launch_kernel(&quantize_kernel<uint16_t, Eight16>, grid, block,
                              0, stream, static_cast<const uint16_t*>(x),
                              words, scales, chunks)
              : launch_kernel(&quantize_kernel<float, Eight32>, grid, block, 0,
                              stream, static_cast<const float*>(x), words,
                              scales, chunks);
}

hipError_t launch_mxfp4_dequantize(const uint8_t* codes,
                                   const uint8_t* scales, void* out, int bf16,
                                   size_t n, hipStream_t stream) {
  if (n % 32 != 0) return hipErrorInvalidValue;
  if (n == 0) return hipSuccess;
  const size_t chunks = n / 8;
  const auto* words = reinterpret_cast<const uint32_t*>(codes);
  const dim3 grid(grid_for(chunks)), block(kThreads);
  return bf16 ? launch_kernel(&dequantize_kernel<uint16_t>, grid, block, 0,
                              stream, words, scales,
                              static_cast<uint16_t*>(out), chunks)
              : launch_kernel(&dequantize_kernel<float>, grid, block, 0,
                              stream, words, scales, static_cast<float*>(out),
                              chunks);
}

}  // namespace kiosk
