// mx_rows.hip -- products of a few rows with an MXFP4 weight: the weight goes
// from memory to the matrix instructions once, through registers alone.
//
// A workgroup owns 16 RT weight rows, its waves share K in pieces (macros) of
// 512.  Within a macro a lane takes the four blocks 4g .. 4g+3 of its row (g =
// lane / 16) in four instructions, block 4g+s in instruction s: 64 contiguous
// bytes per lane and one dword of scales, where the order of K would give each
// instruction 64-byte pieces of rows.  The activations are the 16 CT columns of
// the other operand: the digit planes of M rows (column m P + p: mx_gemm.hip
// has the digits), or the rows themselves where they are microscaled.  The
// waves' sums, and the planes', are added through LDS in a fixed order.
//
// Three f32 rows (five bf16) fill one column tile, and each wave makes the
// digits of its own macro (eight elements per lane and row) while its weight
// loads are on their way: one launch, no workspace.  More rows are split first
// by k_mx_split_cols into fragment order, 1 KB per load.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mx_common.hpp"
#include "mx_digits.hpp"
#include "mx_kernels.hpp"
#include "rt_device.hpp"

namespace rt {
namespace {

constexpr int kMacro = 512;  // elements of K in four instructions
constexpr int kMaxWaves(int ct) { return ct == 1 ? 16 : ct == 2 ? 8 : 4; }  // also: sums in LDS stay within 64 KB
constexpr int kPitch = kMacro + 16;  // of a digit column in LDS: 16 columns of a read on disjoint banks
constexpr int kScaleArea = 96;       // scale bytes of up to six rows
constexpr int digit_area(int cols) { return cols * kPitch + kScaleArea; }  // of a wave

enum Src { kF32, kBf16, kFp8, kFp4, kCols };  // kCols: digit columns in fragment order

struct RowsArgs {
  const uint8_t *w, *wscale;
  const void *a;           // f32 / bf16 rows, microscaled elements, or digit columns
  const uint8_t *ascale;   // microscaled: [m][K/32]; digit columns: a dword per macro, tile and lane
  const float *bias;
  void *c;
  int M, N, K, nmac, planes;
};

// Scale bytes of blocks b .. b+3 of a row of kb (b % 4 == 0); past its end 127.
RT_DEV uint32_t scale_dword(const uint8_t *row, int b, int kb) {
  if ((kb & 3) == 0) return b < kb ? *reinterpret_cast<const uint32_t *>(row + b) : 0x7F7F7F7Fu;
  uint32_t v = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) v |= (b + i < kb ? (uint32_t)row[b + i] : 127u) << (8 * i);
  return v;
}

RT_DEV v4i load_block(const uint8_t *p, bool in) { return in ? *reinterpret_cast<const v4i *>(p) : (v4i){0, 0, 0, 0}; }
RT_DEV v4i load_block_nt(const uint8_t *p, bool in) {
  return in ? __builtin_nontemporal_load(reinterpret_cast<const v4i *>(p)) : (v4i){0, 0, 0, 0};
}

template <int SRC, bool TWO, int RT, int CT, class C>
__global__ __launch_bounds__(64 * kMaxWaves(CT)) void k_mx_rows(RowsArgs g) {
  constexpr bool kOwnDigits = SRC == kF32 || SRC == kBf16, kNarrow = SRC == kFp4;
  constexpr int P = SRC == kF32 ? kPlanesF32 : SRC == kBf16 ? kPlanesBf16 : 1;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = (int)threadIdx.x & 63, l16 = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), waves = (int)blockDim.x >> 6;
  const int n0 = (int)blockIdx.x * 16 * RT, kb = g.K / 32;
  const uint8_t *we[RT], *wsr[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const size_t r = (size_t)min(n0 + 16 * i + l16, g.N - 1);
    we[i] = g.w + r * (g.K / 2);
    wsr[i] = g.wscale + r * kb;
  }
  v4f acc[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j) acc[i][j] = (v4f){0.f, 0.f, 0.f, 0.f};
  uint8_t *dig = lds + wave * digit_area(g.M * P), *dsc = dig + g.M * P * kPitch;  // own digits: columns, scales [row][16]
  const int col = min(l16, g.M * P - 1), col_m = col / P, col_p = col % P;  // columns past the last are never added

  for (int t = wave; t < g.nmac; t += waves) {
    const int b0 = 16 * t + 4 * grp;  // this lane's first block
    v4i wq[RT][4];
    uint32_t ws[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
#pragma unroll
      for (int s = 0; s < 4; ++s) wq[i][s] = load_block_nt(we[i] + (size_t)(b0 + s) * 16, b0 + s < kb);
      ws[i] = scale_dword(wsr[i], b0, kb);
    }
    uint32_t as[CT];
    v4i own[kOwnDigits ? 4 : 1][2];
    // the block that logical block (g / 2) or (2 + g / 2) of instruction s is
    const int c0 = 16 * t + 4 * (grp >> 1), c1 = c0 + 8, half = 16 * (grp & 1);
    if constexpr (kOwnDigits) {
      for (int m = 0; m < g.M; ++m) {
        float v[8] = {};
        const int k0 = kMacro * t + 8 * lane;
        if (k0 < g.K) {
          if constexpr (SRC == kF32) load8(static_cast<const float *>(g.a) + (size_t)m * g.K + k0, v);
          else load8(static_cast<const uint16_t *>(g.a) + (size_t)m * g.K + k0, v);
        }
        uint2 q[P];
        const uint32_t b = digits8<P>(v, q);
#pragma unroll
        for (int p = 0; p < P; ++p) *reinterpret_cast<uint2 *>(dig + (m * P + p) * kPitch + 8 * lane) = q[p];
        if ((lane & 3) == 0) dsc[m * 16 + (lane >> 2)] = (uint8_t)b;
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint8_t *d = dig + col * kPitch + half;
        own[s][0] = *reinterpret_cast<const v4i *>(d + (4 * (grp >> 1) + s) * 32);
        own[s][1] = *reinterpret_cast<const v4i *>(d + (4 * (grp >> 1) + 8 + s) * 32);
      }
      const uint32_t sc = *reinterpret_cast<const uint32_t *>(dsc + col_m * 16 + 4 * grp);
      as[0] = sc - 0x01010101u * kPlaneShift * col_p;  // no borrow: a byte is at least 20
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    } else {
#pragma unroll
      for (int j = 0; j < CT; ++j) {
        if constexpr (SRC == kCols) as[j] = reinterpret_cast<const uint32_t *>(g.ascale)[((size_t)t * CT + j) * 64 + lane];
        else as[j] = scale_dword(g.ascale + (size_t)min(16 * j + l16, g.M - 1) * kb, b0, kb);
      }
    }
    auto mul = [&](auto sc) __attribute__((always_inline)) {
      constexpr int s = decltype(sc)::value;
#pragma unroll
      for (int j = 0; j < CT; ++j) {
        v4i x, y = {0, 0, 0, 0};
        if constexpr (kOwnDigits) {
          x = own[s][0], y = own[s][1];
        } else if constexpr (SRC == kCols) {
          const uint8_t *d = static_cast<const uint8_t *>(g.a) + (((size_t)t * CT + j) * 4 + s) * 2048 + lane * 16;
          x = *reinterpret_cast<const v4i *>(d), y = *reinterpret_cast<const v4i *>(d + 1024);
        } else {
          const uint8_t *d = static_cast<const uint8_t *>(g.a) + (size_t)min(16 * j + l16, g.M - 1) * (kNarrow ? g.K / 2 : g.K);
          if constexpr (kNarrow) {
            x = load_block(d + (size_t)(b0 + s) * 16, b0 + s < kb);
          } else {
            x = load_block(d + (size_t)(c0 + s) * 32 + half, c0 + s < kb);
            y = load_block(d + (size_t)(c1 + s) * 32 + half, c1 + s < kb);
          }
        }
        v8i bv = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}, up = bv;
        if constexpr (TWO) {
#pragma unroll
          for (int i = 0; i < 8; ++i) up[i] = (int)fp8_upper((uint32_t)bv[i]), bv[i] ^= up[i];
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          const v8i wv = {wq[i][s][0], wq[i][s][1], wq[i][s][2], wq[i][s][3], 0, 0, 0, 0};
          if constexpr (TWO)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, up, acc[i][j], 4, 0, s, (int)ws[i], s, (int)as[j]);
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, bv, acc[i][j], 4, kNarrow ? 4 : 0, s, (int)ws[i], s, (int)as[j]);
        }
      }
    };
    mul(IntC<0>{});
    mul(IntC<1>{});
    mul(IntC<2>{});
    mul(IntC<3>{});
  }

  // [wave][tile][lane] of four weight rows each
  __syncthreads();  // the digits' LDS is free
  float *red = reinterpret_cast<float *>(lds);
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j)
      *reinterpret_cast<v4f *>(red + (((wave * RT + i) * CT + j) * 64 + lane) * 4) = acc[i][j];
  __syncthreads();
  const int planes = SRC == kCols ? g.planes : P;
  for (int o = (int)threadIdx.x; o < 16 * RT * g.M; o += (int)blockDim.x) {
    const int r = o % (16 * RT), m = o / (16 * RT), n = n0 + r;
    if (n >= g.N) continue;
    float v = 0.f;
    for (int w = 0; w < waves; ++w)
      for (int p = 0; p < planes; ++p) {
        const int col = m * planes + p;
        v += red[(((w * RT + (r >> 4)) * CT + (col >> 4)) * 64 + ((r >> 2) & 3) * 16 + (col & 15)) * 4 + (r & 3)];
      }
    if (g.bias) v += g.bias[n];
    if constexpr (sizeof(C) == 4) static_cast<float *>(g.c)[(size_t)m * g.N + n] = v;
    else static_cast<uint16_t *>(g.c)[(size_t)m * g.N + n] = f32_to_bf16_bits(v);
  }
}

// Digit columns of M rows for k_mx_rows<kCols>: [macro][column tile][instruction][half][lane][16],
// scales a dword per [macro][column tile][lane].  K is filled up to whole macros
// with zeros; columns past M P are left as they are (they reach no output).
template <class T, int P>
__global__ __launch_bounds__(256) void k_mx_split_cols(const T *__restrict__ x, uint8_t *__restrict__ cols,
                                                       uint8_t *__restrict__ scales, int M, int K, int nmac, int CT) {
  const int i = (int)blockIdx.x * 256 + (int)threadIdx.x, per_row = nmac * (kMacro / 8);
  if (i >= M * per_row) return;  // per_row is whole waves
  const int m = i / per_row, k0 = 8 * (i - m * per_row);
  float v[8] = {};
  if (k0 < K) load8(x + (size_t)m * K + k0, v);
  uint2 q[P];
  const uint32_t b = digits8<P>(v, q);
  const int t = k0 / kMacro, blk = (k0 % kMacro) / 32, j = blk >> 2, s = blk & 3;
  const int g = (j & 1) * 2 + ((k0 >> 4) & 1), h = j >> 1;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int col = m * P + p;
    const size_t tile = (size_t)t * CT + (col >> 4);
    *reinterpret_cast<uint2 *>(cols + ((tile * 4 + s) * 2 + h) * 1024 + (g * 16 + (col & 15)) * 16 + (k0 & 8)) = q[p];
    // the lane of logical block j carries its scales
    if ((k0 & 31) == 0) scales[(tile * 64 + j * 16 + (col & 15)) * 4 + s] = (uint8_t)(b == 255 ? 255 : b - kPlaneShift * p);
  }
}

size_t r256(size_t b) { return (b + 255) & ~size_t(255); }

struct RowsPlan {
  bool ok, split;  // served here; activations split first
  int rt, ct, waves;
};
RowsPlan rows_plan(MxAct act, int m, int n, int k) {
  const int planes = act == kMxActF32 ? kPlanesF32 : act == kMxActBf16 ? kPlanesBf16 : 1;
  const int64_t cols = (int64_t)m * planes;
  RowsPlan p{};
  if (cols > 64) return p;
  p.ok = true;
  p.ct = cols <= 16 ? 1 : cols <= 32 ? 2 : 4;
  p.rt = p.ct;
  p.split = planes > 1 && p.ct > 1;
  const int nmac = (k + kMacro - 1) / kMacro;
  const int64_t wgs = (n + 16 * p.rt - 1) / (16 * p.rt);
  // about 16 waves per CU; then as few as give the same number of macros per wave
  int cap = std::min(nmac, kMaxWaves(p.ct));
  if (planes > 1 && !p.split) cap = std::min(cap, 65536 / digit_area((int)cols));
  const int w = (int)std::min<int64_t>(cap, std::max<int64_t>((4096 + wgs - 1) / wgs, 4));
  const int per = (nmac + w - 1) / w;
  p.waves = (nmac + per - 1) / per;
  return p;
}

template <int SRC, bool TWO, class C>
hipError_t rows_launch(const RowsPlan &p, const RowsArgs &g, hipStream_t s) {
  const dim3 grid((unsigned)((g.N + 16 * p.rt - 1) / (16 * p.rt))), block(64 * p.waves);
  const size_t red = (size_t)p.waves * p.rt * p.ct * 1024;
  constexpr int P = SRC == kF32 ? kPlanesF32 : kPlanesBf16;
  const size_t dig = SRC == kF32 || SRC == kBf16 ? (size_t)p.waves * digit_area(g.M * P) : 0;
  const size_t lds = std::max(red, dig);  // at most 64 KB
  void (*kern)(RowsArgs) = nullptr;
  if constexpr (SRC == kF32 || SRC == kBf16) kern = k_mx_rows<SRC, TWO, 1, 1, C>;
  else kern = p.ct == 1 ? k_mx_rows<SRC, TWO, 1, 1, C> : p.ct == 2 ? k_mx_rows<SRC, TWO, 2, 2, C> : k_mx_rows<SRC, TWO, 4, 4, C>;
  hipLaunchKernelGGL(kern, grid, block, lds, s, g);
  return hipGetLastError();
}

}  // namespace

bool mx_rows_ok(MxAct act, int m, int n, int k) { return rows_plan(act, m, n, k).ok; }

size_t mx_rows_workspace_bytes(MxAct act, int m, int n, int k) {
  const RowsPlan p = rows_plan(act, m, n, k);
  const size_t tiles = (size_t)((k + kMacro - 1) / kMacro) * p.ct;
  return p.split ? r256(tiles * 8192) + r256(tiles * 256) : 0;
}

hipError_t launch_mx_rows(MxAct act, const void *a, const void *w, const float *bias, void *c, bool c_bf16, int m,
                          int n, int k, void *ws, hipStream_t s) {
  const RowsPlan p = rows_plan(act, m, n, k);
  const int nmac = (k + kMacro - 1) / kMacro;
  const uint8_t *we = static_cast<const uint8_t *>(w), *ae = static_cast<const uint8_t *>(a);
  RowsArgs g{we, we + (size_t)n * k / 2, a, nullptr, bias, c, m, n, k, nmac, 1};
  if (p.split) {
    uint8_t *cols = static_cast<uint8_t *>(ws), *sc = cols + r256((size_t)nmac * p.ct * 8192);
    const dim3 grid((unsigned)(((int64_t)m * nmac * (kMacro / 8) + 255) / 256)), block(256);
    if (act == kMxActF32)
      hipLaunchKernelGGL((k_mx_split_cols<float, kPlanesF32>), grid, block, 0, s, static_cast<const float *>(a), cols, sc, m, k, nmac, p.ct);
    else
      hipLaunchKernelGGL((k_mx_split_cols<uint16_t, kPlanesBf16>), grid, block, 0, s, static_cast<const uint16_t *>(a), cols, sc, m, k, nmac, p.ct);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    g.a = cols, g.ascale = sc, g.planes = act == kMxActF32 ? kPlanesF32 : kPlanesBf16;
    return rows_launch<kCols, false, float>(p, g, s);
  }
  switch (act) {
    case kMxActF32: return rows_launch<kF32, false, float>(p, g, s);
    case kMxActBf16: return rows_launch<kBf16, false, float>(p, g, s);
    case kMxActFp8:
      g.ascale = ae + (size_t)m * k;
      return c_bf16 ? rows_launch<kFp8, false, uint16_t>(p, g, s) : rows_launch<kFp8, true, float>(p, g, s);
    default:
      g.ascale = ae + (size_t)m * k / 2;
      return c_bf16 ? rows_launch<kFp4, false, uint16_t>(p, g, s) : rows_launch<kFp4, false, float>(p, g, s);
  }
}

}  // namespace rt
