// mx_gemm.hip -- products with an MXFP4 weight on the scaled matrix instructions.
//
//   c[m][n] = sum_k a[m][k] W[n][k] (+ bias[n])
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 128 by 128 x 16 elements as
// they lie in memory, each 32 of K with the two e8m0 scales of its block, and
// adds in f32.  W is the first operand (its row index is the four consecutive
// output registers of a lane: 16-byte stores along n), the activations the second.
//
// What the instruction keeps (measured, random and constructed operands): the
// products of eight consecutive k are aligned to the largest exponent sum among
// them and cut 13 binary places below it; the 16 group sums and the accumulator
// are then added to f32 accuracy (cut at 2^-25 of the largest).  e2m1 times e2m1
// spans 8 places: exact.  e4m3 spans more, so
//   - MXFP8 activations with an f32 result run as two instructions, one on the
//     elements of 2 and above (exponent field 8..15: bit 6 of the byte), one on
//     the rest: products of each span at most 13 places, so every product counts
//     in full.  With a bf16 result one instruction does (its cut gives about
//     5e-6 of the result's norm, bf16's rounding 2e-3).
//   - f32 and bf16 activations run as e4m3 digits on a grid of 1/4, at most 256:
//     13 places, exact.
//
// Digits: rounding to e4m3 keeps 4 significant bits and leaves at most 2^-5 of
// the value's power of two; so with 2^s a block's scale (its largest value in
// [128, 256))
//   q_p = e4m3(round(r_p 2^(5p-s), 1/4)),  r_(p+1) = r_p - q_p 2^(s-5p),  r_0 = x
// five planes hold an f32's 24 bits and three a bf16's 8, down to 2^-30 and
// 2^-20 of the block's largest value.  The remainders are exact in f32.  The
// product is the sum of the planes' products; W is never widened.
#include <hip/hip_runtime.h>

#include "mx_common.hpp"
#include "mx_kernels.hpp"
#include "rt_device.hpp"

namespace rt {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kPlanesF32 = 5, kPlanesBf16 = 3, kPlaneShift = 5;

// Digit planes of activations [rows][k]: plane p at planes + p rows k, e4m3,
// one scale byte per block (that of plane 0; plane p's is 5p less, so it is at
// least 20).  A thread holds eight elements, a block is a quad.
template <class T, int P>
__global__ __launch_bounds__(256) void k_mx_split(const T *__restrict__ x, uint8_t *__restrict__ planes,
                                                  uint8_t *__restrict__ scales, size_t n8) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n8; i += (size_t)gridDim.x * 256) {
    float v[8];
    load8(x + 8 * i, v);
    // plane 0 is below 256: the exponent of the block's largest value less 7
    const int e = (int)(quad_max_u32(absmax8_bits(v)) >> 23);
    const bool bad = e == 255;
    const int b = bad ? 255 : max(e - 7, kPlaneShift * (kPlanesF32 - 1));
    float inv = bad ? 0.f : bits_f32((uint32_t)(254 - b) << 23);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = bad ? 0.f : v[j] * inv;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float t[8];
      constexpr float kQuarters = 3145728.f;  // 1.5 2^21: a sum with it is rounded to 2^-2
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = (v[j] + kQuarters) - kQuarters;
      const uint2 q = fp8x8(t);
      reinterpret_cast<uint2 *>(planes + (size_t)p * 8 * n8)[i] = q;
      if (p + 1 < P) {
        typedef float v2f __attribute__((ext_vector_type(2)));
        const v2f d0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, false), d1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, true);
        const v2f d2 = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, false), d3 = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, true);
        const float d[8] = {d0.x, d0.y, d1.x, d1.y, d2.x, d2.y, d3.x, d3.y};
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (v[j] - d[j]) * 32.f;
      }
    }
    if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)b;
  }
}

struct MxOperand {
  const uint8_t *e, *s;
  size_t plane;  // bytes from one digit plane to the next
  int planes;
};

// Four e8m0 bytes of blocks 4t .. 4t+3 of a row of kb blocks (past its end 127:
// the elements there are zero).
RT_DEV int scale4(const uint8_t *row, int kb, int t) {
  if ((kb & 3) == 0) return *reinterpret_cast<const int *>(row + 4 * t);
  uint32_t v = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) v |= (4 * t + i < kb ? (uint32_t)row[4 * t + i] : 127u) << (8 * i);
  return (int)v;
}

// The elements of 2 and above of four e4m3 bytes (bit 6 is the exponent field's
// top bit), the others zero.
RT_DEV uint32_t fp8_upper(uint32_t x) {
  const uint32_t t = (x >> 6) & 0x01010101u;
  return x & ((t << 8) - t);
}

// One wave per 16 x 16 of c, operands straight from memory.
template <int FA, bool TWO, class C>
__global__ __launch_bounds__(256) void k_mx_gemm_direct(MxOperand a, MxOperand w, const float *__restrict__ bias,
                                                        C *__restrict__ c, int M, int N, int K) {
  const int lane = (int)threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int n0 = ((int)blockIdx.x * 4 + ((int)threadIdx.x >> 6)) * 16, m0 = (int)blockIdx.y * 16;
  const int kb = K / 32, nr = min(n0 + l16, N - 1), mr = min(m0 + l16, M - 1);
  const uint8_t *we = w.e + (size_t)nr * (K / 2), *ws = w.s + (size_t)nr * kb;
  const uint8_t *as = a.s + (size_t)mr * kb;
  v4f acc = {0.f, 0.f, 0.f, 0.f};
  for (int t = 0; t < (kb + 3) / 4; ++t) {
    const v4i zero = {0, 0, 0, 0};
    const int b = 4 * t + g;
    const v4i wq = b < kb ? *reinterpret_cast<const v4i *>(we + (size_t)b * 16) : zero;
    const v8i wv = {wq[0], wq[1], wq[2], wq[3], 0, 0, 0, 0};
    const int wsc = (int)((uint32_t)scale4(ws, kb, t) >> (8 * g)), asc = scale4(as, kb, t) >> (8 * g);
    for (int p = 0; p < a.planes; ++p) {
      v8i av;
      if constexpr (FA == kMxFp8) {
        // a lane's 32 bytes are two half blocks, 64 of K apart
        const uint8_t *ae = a.e + (size_t)p * a.plane + (size_t)mr * K;
        const int b0 = 4 * t + (g >> 1), b1 = b0 + 2;
        const v4i x = b0 < kb ? *reinterpret_cast<const v4i *>(ae + (size_t)b0 * 32 + 16 * (g & 1)) : zero;
        const v4i y = b1 < kb ? *reinterpret_cast<const v4i *>(ae + (size_t)b1 * 32 + 16 * (g & 1)) : zero;
        av = (v8i){x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      } else {
        const v4i x = b < kb ? *reinterpret_cast<const v4i *>(a.e + (size_t)mr * (K / 2) + (size_t)b * 16) : zero;
        av = (v8i){x[0], x[1], x[2], x[3], 0, 0, 0, 0};
      }
      const int ab = (asc & 255) == 255 ? 255 : (asc & 255) - kPlaneShift * p;
      if constexpr (TWO) {
        v8i up;
#pragma unroll
        for (int i = 0; i < 8; ++i) up[i] = (int)fp8_upper((uint32_t)av[i]), av[i] ^= up[i];
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, up, acc, 4, 0, 0, wsc, 0, ab);
      }
      acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, av, acc, 4, FA == kMxFp8 ? 0 : 4, 0, wsc, 0, ab);
    }
  }
  const int row = m0 + l16;
  if (row >= M) return;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int n = n0 + 4 * g + r;
    if (n >= N) continue;
    const float v = acc[r] + (bias ? bias[n] : 0.f);
    if constexpr (sizeof(C) == 4) c[(size_t)row * N + n] = v;
    else c[(size_t)row * N + n] = f32_to_bf16_bits(v);
  }
}

size_t r256(size_t b) { return (b + 255) & ~size_t(255); }
int planes_of(MxAct act) { return act == kMxActF32 ? kPlanesF32 : act == kMxActBf16 ? kPlanesBf16 : 1; }

}  // namespace

size_t mx_gemm_workspace_bytes(MxAct act, int m, int n, int k) {
  if (act == kMxActFp8 || act == kMxActFp4) return 256;
  return r256((size_t)planes_of(act) * m * k) + r256((size_t)m * (k / 32));
}

hipError_t launch_mx_gemm(MxAct act, const void *a, const void *w, const float *bias, void *c, bool c_bf16, int m,
                          int n, int k, void *ws, hipStream_t s) {
  const uint8_t *we = static_cast<const uint8_t *>(w);
  const MxOperand W{we, we + (size_t)n * k / 2, 0, 1};
  MxOperand A;
  const size_t mk = (size_t)m * k;
  if (act == kMxActF32 || act == kMxActBf16) {
    uint8_t *pl = static_cast<uint8_t *>(ws), *sc = pl + r256(planes_of(act) * mk);
    const dim3 g((unsigned)((mk / 8 + 255) / 256 < 65536 ? (mk / 8 + 255) / 256 : 65536)), b(256);
    if (act == kMxActF32)
      hipLaunchKernelGGL((k_mx_split<float, kPlanesF32>), g, b, 0, s, static_cast<const float *>(a), pl, sc, mk / 8);
    else
      hipLaunchKernelGGL((k_mx_split<uint16_t, kPlanesBf16>), g, b, 0, s, static_cast<const uint16_t *>(a), pl, sc, mk / 8);
    A = {pl, sc, mk, planes_of(act)};
  } else {
    const uint8_t *ae = static_cast<const uint8_t *>(a);
    A = {ae, ae + mx_elem_bytes(act == kMxActFp8 ? kMxFp8 : kMxFp4, mk), 0, 1};
  }
  const dim3 grid((n + 63) / 64, (m + 15) / 16), block(256);
  float *cf = static_cast<float *>(c);
  uint16_t *ch = static_cast<uint16_t *>(c);
  if (act == kMxActFp4) {
    if (c_bf16) hipLaunchKernelGGL((k_mx_gemm_direct<kMxFp4, false, uint16_t>), grid, block, 0, s, A, W, bias, ch, m, n, k);
    else hipLaunchKernelGGL((k_mx_gemm_direct<kMxFp4, false, float>), grid, block, 0, s, A, W, bias, cf, m, n, k);
  } else if (act == kMxActFp8) {
    if (c_bf16) hipLaunchKernelGGL((k_mx_gemm_direct<kMxFp8, false, uint16_t>), grid, block, 0, s, A, W, bias, ch, m, n, k);
    else hipLaunchKernelGGL((k_mx_gemm_direct<kMxFp8, true, float>), grid, block, 0, s, A, W, bias, cf, m, n, k);
  } else {
    hipLaunchKernelGGL((k_mx_gemm_direct<kMxFp8, false, float>), grid, block, 0, s, A, W, bias, cf, m, n, k);
  }
  return hipGetLastError();
}

}  // namespace rt
