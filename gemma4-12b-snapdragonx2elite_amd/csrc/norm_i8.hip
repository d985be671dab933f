// Row norms that leave int8: the rmsnorm (or the residual normadd and the
// rmsnorm of the new residual) of each row of [M][D], quantized per row for
// the int8 GEMMs in the same launch.
//
//   n  = x * inv(x) * w,  inv(v) = 1 / sqrt(mean(v^2) + 1e-6)
//   h' = (h + n) * sc                    (with a residual; else y = n)
//   y  = h' * inv(h') * w2
//   sa = max(max|y| / 127, 1e-12),  A = clamp(rint(y / sa), -127, 127)
//
// vk/pre_norm.comp:9-13, vk/pre_na.comp:9-14 and vk/cast_i8.comp:11-19 of the
// reference run as three dispatches with y in memory between them.
#include "q4mi_common.h"

namespace q4 {

// 8 values of a row as fp32: chunk c of thread t. VEC: the 8 consecutive
// elements from 8 (c NT + t) on, in 16-byte loads; else the elements
// (8 c + e) NT + t, one load each (rows of any length and alignment).
template <int NT, bool VEC>
__device__ inline int ni_index(int c, int e) {
  return VEC ? 8 * (c * NT + (int)threadIdx.x) + e : (8 * c + e) * NT + (int)threadIdx.x;
}
template <int NT, bool VEC, int XT>
__device__ inline void ni_load(const void* p, int c, int D, float (&v)[8]) {
  if constexpr (VEC) {
    const int i = ni_index<NT, VEC>(c, 0);
    if (i >= D) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    } else if constexpr (XT == Q4_DT_F16) {
      const v4u u = *reinterpret_cast<const v4u*>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[2 * k] = h2f((uint16_t)(u[k] & 0xFFFFu));
        v[2 * k + 1] = h2f((uint16_t)(u[k] >> 16));
      }
    } else {
      const v4f a = *reinterpret_cast<const v4f*>(reinterpret_cast<const float*>(p) + i);
      const v4f b = *reinterpret_cast<const v4f*>(reinterpret_cast<const float*>(p) + i + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = a[k];
        v[4 + k] = b[k];
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = ni_index<NT, VEC>(c, e);
      if constexpr (XT == Q4_DT_F16) v[e] = i < D ? h2f(reinterpret_cast<const uint16_t*>(p)[i]) : 0.0f;
      else v[e] = i < D ? reinterpret_cast<const float*>(p)[i] : 0.0f;
    }
  }
}

// Sum of a and maximum of b over the workgroup, the same bits in every
// thread; red: 2 NT / 64 floats that no wave still reads.
template <int NT>
__device__ inline void ni_reduce(float& a, float& b, float* red) {
  constexpr int NW = NT / 64;
  a = reduce64<false>(a);
  b = reduce64<true>(b);
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = a;
    red[NW + (threadIdx.x >> 6)] = b;
  }
  __syncthreads();
  a = red[0];
  b = red[NW];
#pragma unroll
  for (int i = 1; i < NW; ++i) {
    a += red[i];
    b = fmaxf(b, red[NW + i]);
  }
}

// One row per workgroup, every operand in registers (NC chunks of 8 values
// per thread) up to D 16384; past it 1024 threads leave 128 registers each,
// and the form with the residual, 128 values and more, spills 49 to 98. The
// largest |y| is the largest |h' w2| times inv(h'), so it is reduced with the
// sum of squares: one barrier per norm. All loads are issued before the first
// reduction. Bound by memory for many rows (2048 rows
// of 3840 with fp16 x and the residual: 86.5 MB in 17 us, 5 TB/s, the rate of a
// copy, where part of it is in the cache; 22.7 us on cold data), by the launch
// and one round trip of loads for few (one row 3.2 us, 128 rows 4.2 us).
template <int NT, int NC, bool VEC, bool ADD, int XT>
__global__ void __launch_bounds__(NT) norm_i8_kernel(const void* __restrict__ x, const float* __restrict__ w,
                                                     float* __restrict__ h, int D, float sc,
                                                     const float* __restrict__ w2, int8_t* __restrict__ A,
                                                     float* __restrict__ sa) {
  __shared__ float red[2][2 * NT / 64];
  const long row = blockIdx.x;
  x = reinterpret_cast<const char*>(x) + row * D * (XT == Q4_DT_F16 ? 2 : 4);
  A += row * D;
  float v[NC][8], wv[NC][8], w2v[ADD ? NC : 1][8], hv[ADD ? NC : 1][8];
#pragma unroll
  for (int c = 0; c < NC; ++c) ni_load<NT, VEC, XT>(x, c, D, v[c]);
  if constexpr (ADD) {
    h += row * D;
#pragma unroll
    for (int c = 0; c < NC; ++c) ni_load<NT, VEC, Q4_DT_F32>(h, c, D, hv[c]);
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) ni_load<NT, VEC, Q4_DT_F32>(w, c, D, wv[c]);
  if constexpr (ADD) {
#pragma unroll
    for (int c = 0; c < NC; ++c) ni_load<NT, VEC, Q4_DT_F32>(w2, c, D, w2v[c]);
  }
  float ss = 0.0f, mx = 0.0f;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ss = fmaf(v[c][e], v[c][e], ss);
      if constexpr (!ADD) mx = fmaxf(mx, fabsf(v[c][e] * wv[c][e]));
    }
  ni_reduce<NT>(ss, mx, red[0]);
  float inv = inv_rms(ss, D);
  if constexpr (ADD) {
    float s2 = 0.0f;
    mx = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float n = __fmul_rn(__fmul_rn(v[c][e], inv), wv[c][e]);
        const float u = __fmul_rn(__fadd_rn(hv[c][e], n), sc);
        v[c][e] = u;
        wv[c][e] = w2v[c][e];
        s2 = fmaf(u, u, s2);  // elements past the row are 0
        mx = fmaxf(mx, fabsf(u * w2v[c][e]));
      }
      if constexpr (VEC) {
        const int i = ni_index<NT, VEC>(c, 0);
        if (i < D) {
          *reinterpret_cast<v4f*>(h + i) = v4f{v[c][0], v[c][1], v[c][2], v[c][3]};
          *reinterpret_cast<v4f*>(h + i + 4) = v4f{v[c][4], v[c][5], v[c][6], v[c][7]};
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = ni_index<NT, VEC>(c, e);
          if (i < D) h[i] = v[c][e];
        }
      }
    }
    ni_reduce<NT>(s2, mx, red[1]);
    inv = inv_rms(s2, D);
  }
  // the quantizer's rounding: IEEE divisions, rint to even, clamp (a NaN becomes -127, as there)
  const float s = fmaxf(__fdiv_rn(mx * inv, 127.0f), 1e-12f);
  if (threadIdx.x == 0) sa[row] = s;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = __fmul_rn(__fmul_rn(v[c][e], inv), wv[c][e]);
      b[e] = (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(y, s)), -127.0f), 127.0f) & 0xFFu;
    }
    if constexpr (VEC) {
      const int i = ni_index<NT, VEC>(c, 0);
      if (i < D)
        *reinterpret_cast<v2u*>(A + i) = v2u{b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24,
                                             b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = ni_index<NT, VEC>(c, e);
        if (i < D) A[i] = (int8_t)b[e];
      }
    }
  }
}

constexpr int NI_MAX_D = 32768;      // 1024 threads of four chunks
constexpr int NI_MAX_M = 1 << 22;    // a launch holds fewer than 2^32 threads

template <int NT, int NC, bool ADD, int XT>
static void ni_launch(const void* x, const float* w, float* h, int D, int M, float sc, const float* w2, int8_t* A,
                      float* sa, bool vec, hipStream_t st) {
  if (vec)
    hipLaunchKernelGGL((norm_i8_kernel<NT, NC, true, ADD, XT>), dim3(M), dim3(NT), 0, st, x, w, h, D, sc, w2, A, sa);
  else
    hipLaunchKernelGGL((norm_i8_kernel<NT, NC, false, ADD, XT>), dim3(M), dim3(NT), 0, st, x, w, h, D, sc, w2, A, sa);
}
template <bool ADD, int XT>
static void ni_rows(const void* x, const float* w, float* h, int D, int M, float sc, const float* w2, int8_t* A,
                    float* sa, hipStream_t st) {
  auto al = [](const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; };
  const bool vec = D % 8 == 0 && al(x, 16) && al(w, 16) && al(A, 8) && (!ADD || (al(h, 16) && al(w2, 16)));
  // threads by row length, us per launch among others at 1 / 128 / 2048 rows of fp32 with the residual:
  //   D  2000: 256 x 1 chunk 3.0 / 3.8 / 14.0, 512 x 1 3.0 / 3.9 / 14.8, 1024 x 1 3.5 / 4.4 / 21.0
  //   D  3840: 512 x 1 3.5 / 4.6 / 24.8, 256 x 2 3.6 / 4.7 / 25.1, 128 x 4 4.3 / 5.5 / 28.4, 1024 x 1 4.0 / 5.1 / 28.0
  //   D  5120: 512 x 2 4.0 / 5.3 / 32.4, 256 x 4 4.2 / 5.5 / 32.2, 1024 x 1 4.4 / 5.7 / 34.3
  //   D 15360: 512 x 4 6.9 / 12.6 / 97.7, 1024 x 2 7.0 / 12.8 / 99.3
  // and single-element accesses of the same rows: 14.2 at D 2000, 25.7 at 3840, 42.7 at 5120, 106 at 15360 (2048 rows);
  // past D 16384 (4 chunks of 1024 threads, the residual form spilling), fp16 x, us per call from Python: D 20000
  // 13.6 / 21.5 / 254 (single-element accesses, D 20001: 493 at 2048 rows), D 32768 17.6 / 30.3 / 322 (765 at 32767);
  // without the residual D 32768 87.5 at 2048 rows
  if (D <= 2048) ni_launch<256, 1, ADD, XT>(x, w, h, D, M, sc, w2, A, sa, vec, st);
  else if (D <= 4096) ni_launch<512, 1, ADD, XT>(x, w, h, D, M, sc, w2, A, sa, vec, st);
  else if (D <= 8192) ni_launch<512, 2, ADD, XT>(x, w, h, D, M, sc, w2, A, sa, vec, st);
  else if (D <= 16384) ni_launch<512, 4, ADD, XT>(x, w, h, D, M, sc, w2, A, sa, vec, st);
  else ni_launch<1024, 4, ADD, XT>(x, w, h, D, M, sc, w2, A, sa, vec, st);
}

// Whether n bytes of rows that are written, the weights w and the scales sa share no byte.
static bool ni_apart(const void* rows, size_t n, const float* w, int D, const float* sa, int M) {
  return !overlap(rows, n, w, (size_t)D * 4) && !overlap(rows, n, sa, (size_t)M * 4) &&
         !overlap(w, (size_t)D * 4, sa, (size_t)M * 4);
}

}  // namespace q4

using namespace q4;

extern "C" {

int q4_pre_rmsnorm_i8(const float* x, const float* w, int8_t* A, float* sa, int D, int M, void* stream) {
  clear_error();
  Q4_ARG(x && w && A && sa, "null pointer");
  Q4_ARG(D > 0 && D <= NI_MAX_D && M > 0 && M < NI_MAX_M, "bad sizes D=%d M=%d (D up to %d, M below %d)", D, M,
         NI_MAX_D, NI_MAX_M);
  Q4_ARG(!overlap(x, (size_t)M * D * 4, A, (size_t)M * D), "A must not overlap x");
  Q4_ARG(ni_apart(A, (size_t)M * D, w, D, sa, M) && !overlap(sa, (size_t)M * 4, x, (size_t)M * D * 4),
         "A and sa must not overlap each other, x or w");
  ni_rows<false, Q4_DT_F32>(x, w, nullptr, D, M, 1.0f, nullptr, A, sa, as_stream(stream));
  Q4_LAUNCHED("pre_rmsnorm_i8");
  return Q4_OK;
}

int q4_pre_normadd_rmsnorm_i8(const void* x, int x_dtype, const float* w, float* h, int D, int M, float scale,
                              const float* w2, int8_t* A, float* sa, void* stream) {
  clear_error();
  Q4_ARG(x && w && h && w2 && A && sa, "null pointer");
  Q4_ARG(D > 0 && D <= NI_MAX_D && M > 0 && M < NI_MAX_M, "bad sizes D=%d M=%d (D up to %d, M below %d)", D, M,
         NI_MAX_D, NI_MAX_M);
  Q4_ARG(x_dtype == Q4_DT_F32 || x_dtype == Q4_DT_F16, "bad x_dtype");
  const size_t n = (size_t)M * D;
  Q4_ARG(!overlap(x, n * (x_dtype == Q4_DT_F16 ? 2 : 4), h, n * 4), "x must not overlap h");
  Q4_ARG(!overlap(x, n * (x_dtype == Q4_DT_F16 ? 2 : 4), A, n) && !overlap(h, n * 4, A, n), "A must not overlap x or h");
  Q4_ARG(ni_apart(A, n, w, D, sa, M) && ni_apart(A, n, w2, D, sa, M) && ni_apart(h, n * 4, w, D, sa, M) &&
             ni_apart(h, n * 4, w2, D, sa, M) && !overlap(sa, (size_t)M * 4, x, n * (x_dtype == Q4_DT_F16 ? 2 : 4)),
         "h, A and sa must not overlap each other, x, w or w2");
  const float sc = scale == 0.0f ? 1.0f : scale;
  if (x_dtype == Q4_DT_F16) ni_rows<true, Q4_DT_F16>(x, w, h, D, M, sc, w2, A, sa, as_stream(stream));
  else ni_rows<true, Q4_DT_F32>(x, w, h, D, M, sc, w2, A, sa, as_stream(stream));
  Q4_LAUNCHED("pre_normadd_rmsnorm_i8");
  return Q4_OK;
}

}  // extern "C"
