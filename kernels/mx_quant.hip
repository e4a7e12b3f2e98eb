// Rows to microscaled codes and scales (formats and rounding: mx.h), and back.
//
// Bound by bytes.  A thread has a whole block: its largest magnitude and its codes need no other
// lane, and it stores 16 bytes of them.  (Eight values a thread, the scale by two exchanges,
// took 84 us instead of 50 for 8192 x 14336, four bytes and quarters of scales a store.)  50 us
// of 235 MB of x and 62 MB of codes, 5.9 TB/s, are 51 to 53 where x comes from memory and 66 to
// 78 behind a launch whose own 235 MB of results are still on their way there; 6 bits 57.  The
// products read rows of whole tiles of 256 inputs or pairs of them, zeros behind the last, and
// 6-bit codes as two planes, the first 16 bytes of each block's 24 and the other 8, a tile's in
// the order of mx::place_of: either reaches LDS in pieces of 16 bytes.

#include "mx_product.h"
#include "mx_round.h"

namespace {

// Scale bytes to rows of whole tiles, 256 a workgroup
DEVINLINE void pad_scales(const MxPad& pad, int blocks, int in_row, long workgroup) {
  const long i = workgroup * 256 + threadIdx.x, row = i / in_row;
  if (row >= pad.rows) return;
  const int b = (int)(i - row * in_row);
  pad.to[i] = b < blocks ? pad.from[row * blocks + b] : 0;
}
__global__ __launch_bounds__(256) void mx_pad_scales_kernel(const MxPad pad, const int blocks,
                                                            const int in_row) {
  pad_scales(pad, blocks, in_row, blockIdx.x);
}

// plane0 [rows, stride0], plane1 [rows, stride0 / 2] or null (a block's bytes one after the
// other, or 4 bits), scales [rows, in_row]; a row is in_row blocks, zeros past its `blocks`.
template <typename T, int BITS>
__global__ __launch_bounds__(256) void mx_rows_kernel(
    unsigned char* __restrict__ plane0, unsigned char* __restrict__ plane1,
    unsigned char* __restrict__ scales, const T* __restrict__ x, const long all, const long pitch,
    const int blocks, const int in_row, const long stride0, const bool aligned, const MxPad pad,
    const long pads) {   // workgroups that pad, behind the others
  if (blockIdx.x >= gridDim.x - pads) {
    pad_scales(pad, blocks, in_row, blockIdx.x - (gridDim.x - pads));
    return;
  }
  // blocks from here on, of rows from the first one's on: 32 bits do
  const long base = (long)blockIdx.x * 256, row0 = base / in_row;
  if (base + threadIdx.x >= all) return;
  const unsigned at = (unsigned)(base - row0 * in_row) + threadIdx.x, r = at / (unsigned)in_row;
  const long row = row0 + r;
  const int b = at - r * in_row;
  mx::Block<T> v{};
  if (b < blocks) {
    const T* from = x + row * pitch + (long)b * 32;
    if (aligned) {
#pragma unroll
      for (int q = 0; q < mx::Block<T>::kPieces; ++q)
        v.v[q] = reinterpret_cast<const mx::i32x4_t*>(from)[q];
    } else {
      T one[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) one[i] = from[i];
      __builtin_memcpy(&v, one, sizeof(v));
    }
  }
  unsigned byte;
  mx::i32x8_t c = mx::rounded<BITS>(v, byte);
  if (byte == 255) c = mx::i32x8_t{};
  scales[row * in_row + b] = (unsigned char)byte;
  if constexpr (BITS == 4) {
    *reinterpret_cast<mx::i32x4_t*>(plane0 + row * stride0 + b * 16) =
        mx::i32x4_t{c[0], c[1], c[2], c[3]};
  } else if (plane1 != nullptr) {
    *reinterpret_cast<mx::i32x4_t*>(plane0 + row * stride0 + b * 16) =
        mx::i32x4_t{c[0], c[1], c[2], c[3]};
    *reinterpret_cast<mx::i32x2_t*>(plane1 + row * (stride0 / 2) + b / 8 * 64 +
                                    mx::place_of(b % 8) * 8) = mx::i32x2_t{c[4], c[5]};
  } else {
    int* to = reinterpret_cast<int*>(plane0 + row * stride0 + b * 24);
#pragma unroll
    for (int i = 0; i < 6; ++i) to[i] = c[i];
  }
}

constexpr int kEach = 4;   // pieces of eight values of a thread, all asked for at once

// Eight values a piece, blocks one after the other.
template <typename T, int BITS>
__global__ __launch_bounds__(256) void mx_values_kernel(T* __restrict__ y,
                                                        const unsigned char* __restrict__ codes,
                                                        const unsigned char* __restrict__ scales,
                                                        const long pieces) {
  const long base = (long)blockIdx.x * (256 * kEach) + threadIdx.x;
  unsigned long long u[kEach];
  unsigned byte[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const long at = base + e * 256;
    if (at < pieces) {
      if constexpr (BITS == 4) {
        u[e] = reinterpret_cast<const unsigned*>(codes)[at];
      } else {
        const unsigned short* from = reinterpret_cast<const unsigned short*>(codes) + at * 3;
        u[e] = from[0] | (unsigned long long)from[1] << 16 | (unsigned long long)from[2] << 32;
      }
      byte[e] = scales[at / 4];
    }
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const long at = base + e * 256;
    if (at >= pieces) break;
    const float scale = mx::scale_value(byte[e]);
    float v[8];
    if constexpr (BITS == 4) {
      typedef __attribute__((ext_vector_type(2))) float f32x2_t;
      const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((unsigned)u[e], 1.f, 0);
      const f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((unsigned)u[e], 1.f, 1);
      const f32x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((unsigned)u[e], 1.f, 2);
      const f32x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((unsigned)u[e], 1.f, 3);
      const float w[8] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = w[i] * scale;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = mx::value6((unsigned)(u[e] >> (6 * i)) & 63) * scale;
    }
#pragma unroll
    for (int h = 0; h < 8 / Vec16<T>::kElems; ++h) {
      Vec16<T> o;
#pragma unroll
      for (int i = 0; i < Vec16<T>::kElems; ++i)
        o.data[i] = ScalarOps<T>::from_f32(v[h * Vec16<T>::kElems + i]);
      store16(y + at * 8 + h * Vec16<T>::kElems, o);
    }
  }
}

}  // namespace

template <typename T>
void launch_mx_rows(unsigned char* plane0, unsigned char* plane1, unsigned char* scales, const T* x,
                    long rows, long pitch, int K, int padded, int bits, const MxPad& pad,
                    hipStream_t stream) {
  const int in_row = padded / 32;
  const long all = rows * in_row, pads = (pad.rows * in_row + 255) / 256;
  const bool aligned = reinterpret_cast<uintptr_t>(x) % 16 == 0 && pitch * sizeof(T) % 16 == 0;
  const long stride0 = bits == 4 || plane1 != nullptr ? padded / 2 : padded / 4 * 3;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((all + 255) / 256 + pads), dim3(256), 0, stream, plane0, plane1,
                       scales, x, all, pitch, K / 32, in_row, stride0, aligned, pad, pads);
  };
  if (bits == 4) go(mx_rows_kernel<T, 4>);
  else go(mx_rows_kernel<T, 6>);
}

template <typename T>
void launch_mx_values(T* y, const unsigned char* codes, const unsigned char* scales, long values,
                      int bits, hipStream_t stream) {
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((values / 8 + 256 * kEach - 1) / (256 * kEach)), dim3(256), 0,
                       stream, y, codes, scales, values / 8);
  };
  if (bits == 4) go(mx_values_kernel<T, 4>);
  else go(mx_values_kernel<T, 6>);
}

void launch_mx_pad_scales(const MxPad& pad, int K, int padded, hipStream_t stream) {
  const int in_row = padded / 32;
  hipLaunchKernelGGL(mx_pad_scales_kernel, dim3((pad.rows * in_row + 255) / 256), dim3(256), 0, stream,
                     pad, K / 32, in_row);
}

#define MX_TYPES(T)                                                                              \
  template void launch_mx_rows<T>(unsigned char*, unsigned char*, unsigned char*, const T*, long, \
                                  long, int, int, int, const MxPad&, hipStream_t);               \
  template void launch_mx_values<T>(T*, const unsigned char*, const unsigned char*, long, int,   \
                                    hipStream_t);
MX_TYPES(__hip_bfloat16)
MX_TYPES(__half)
MX_TYPES(float)
