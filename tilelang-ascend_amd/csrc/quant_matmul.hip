// 8-bit matrix product with a scale for each token and each output channel.
//
//   out[m, n] = (sum_k x[m, k] w[n, k]) * sx[m] * sw[n] + bias[n]
//
// x [M, K] and w [N, K] are int8 rows as the row quantiser writes them (quant.hip), sx and sw its fp32 row scales.
// The sums are int32 and exact: |x w| <= 2^14 and K <= 131071, so no sum passes 2^31.  The sum is then rounded to
// fp32 (half a step, 2^-24), scaled and biased in fp32 and rounded once to the output type.
#include "common.hpp"

namespace dsa {

enum QmmOut : int { kQmmBf16 = 1, kQmmFp16 = 2, kQmmFp32 = 3 };

struct QmmArgs {
  const uint8_t* x;   // [M, K]
  const uint8_t* w;   // [N, K]
  const float* sx;    // [M]
  const float* sw;    // [N]
  const float* bias;  // [N] or null
  void* out;          // [M, N]
  int M, N, K;
};

// i32 16x16 += A 16x64 B 64x16: lane (r = lane & 15, g = lane >> 4) gives row r of A and column r of B,
// k = 16 g .. 16 g + 15, and holds rows 4 g .. 4 g + 3 of column r of the result.
__device__ __forceinline__ i32x4 qmm_mfma(const u32x4& a, const u32x4& b, const i32x4& c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

template <int kOut>
__device__ __forceinline__ void qmm_store1(void* out, int64_t at, float v) {
  if constexpr (kOut == kQmmFp32) static_cast<float*>(out)[at] = v;
  else if constexpr (kOut == kQmmBf16) static_cast<__bf16*>(out)[at] = (__bf16)v;
  else static_cast<_Float16*>(out)[at] = (_Float16)v;
}

// Four consecutive elements, on their own width.
template <int kOut>
__device__ __forceinline__ void qmm_store4(void* out, int64_t at, const float (&v)[4]) {
  if constexpr (kOut == kQmmFp32) {
    *reinterpret_cast<f32x4*>(static_cast<float*>(out) + at) = f32x4{v[0], v[1], v[2], v[3]};
  } else if constexpr (kOut == kQmmBf16) {
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(out) + at) =
        u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
  } else {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<f16x4*>(static_cast<_Float16*>(out) + at) =
        f16x4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
  }
}

// Any sizes and any alignment: 128 x 128 of the output a workgroup, 64 x 64 a wave, k in steps of 64 through two
// LDS stages.  A row's 16-byte chunks are read where they lie (byte aligned); the chunk that K ends in is
// read by bytes.  LDS rows hold 4 chunks; chunk c of row r lies at c ^ 2 ((r >> 3) & 1), so that the 32 chunks a
// half wave reads at once (16 rows, two chunks) fall on distinct banks.
constexpr int kQmmTile = 128;
constexpr int kQmmStep = 64;

__device__ __forceinline__ u32x4 qmm_chunk(const uint8_t* row, int k, int K) {
  u32x4 v = {0, 0, 0, 0};
  if (k + 16 <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else {
    for (int i = 0; k + i < K; ++i) v[i >> 2] |= (uint32_t)row[k + i] << (8 * (i & 3));
  }
  return v;
}

template <int kOut>
__global__ __launch_bounds__(256, 2) void qmm_tile_kernel(QmmArgs a) {
  __shared__ __align__(16) uint8_t lds[2][2][kQmmTile * kQmmStep];  // stage, operand (w, x)
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int r = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.y * kQmmTile, n0 = blockIdx.x * kQmmTile;
  const int wn = (wave & 1) * 64, wm = (wave >> 1) * 64;

  // Thread t stages chunks t & 3 of rows t / 4 and t / 4 + 64; rows past the edge repeat the last one.
  const uint8_t* src[2][2];
  int dst[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = tid / 4 + 64 * j;
    src[0][j] = a.w + (int64_t)min(n0 + row, a.N - 1) * a.K;
    src[1][j] = a.x + (int64_t)min(m0 + row, a.M - 1) * a.K;
    dst[j] = row * kQmmStep + 16 * ((tid & 3) ^ (2 * ((row >> 3) & 1)));
  }
  u32x4 reg[2][2];
  auto load = [&](int k0) {
    const int k = k0 + 16 * (tid & 3);
    if (k0 + kQmmStep <= a.K) {
#pragma unroll
      for (int o = 0; o < 2; ++o)
#pragma unroll
        for (int j = 0; j < 2; ++j) __builtin_memcpy(&reg[o][j], src[o][j] + k, 16);
    } else {
#pragma unroll
      for (int o = 0; o < 2; ++o)
#pragma unroll
        for (int j = 0; j < 2; ++j) reg[o][j] = qmm_chunk(src[o][j], k, a.K);
    }
  };
  auto put = [&](int st) {
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int j = 0; j < 2; ++j) *reinterpret_cast<u32x4*>(&lds[st][o][dst[j]]) = reg[o][j];
  };
  i32x4 acc[4][4];  // [n block][m block]
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

  const int off = r * kQmmStep + 16 * (g ^ (2 * ((r >> 3) & 1)));
  const int steps = (a.K + kQmmStep - 1) / kQmmStep;
  load(0);
  put(0);
  for (int s = 0; s < steps; ++s) {
    __syncthreads();
    if (s + 1 < steps) load((s + 1) * kQmmStep);
    const uint8_t *lw = lds[s & 1][0] + wn * kQmmStep + off, *lx = lds[s & 1][1] + wm * kQmmStep + off;
    u32x4 wv[4], xv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) wv[i] = *reinterpret_cast<const u32x4*>(lw + i * 16 * kQmmStep);
#pragma unroll
    for (int i = 0; i < 4; ++i) xv[i] = *reinterpret_cast<const u32x4*>(lx + i * 16 * kQmmStep);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = qmm_mfma(wv[i], xv[j], acc[i][j]);
    // The other stage's reads were done before the barrier above.
    if (s + 1 < steps) put((s + 1) & 1);
  }

  const bool vec = (a.N & 3) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int m = m0 + wm + 16 * j + r;
    if (m >= a.M) continue;
    const float sx = a.sx[m];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + wn + 16 * i + 4 * g;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int ne = min(n + e, a.N - 1);
        v[e] = (float)acc[i][j][e] * sx * a.sw[ne];
        if (a.bias) v[e] += a.bias[ne];
      }
      const int64_t at = (int64_t)m * a.N + n;
      if (vec) {
        if (n < a.N) qmm_store4<kOut>(a.out, at, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < a.N) qmm_store1<kOut>(a.out, at + e, v[e]);
      }
    }
  }
}

template <int kOut>
static hipError_t qmm_launch(const QmmArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.N + kQmmTile - 1) / kQmmTile), (unsigned)((a.M + kQmmTile - 1) / kQmmTile));
  hipLaunchKernelGGL((qmm_tile_kernel<kOut>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

size_t quant_matmul_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

// Caller validated: 1 <= K <= 131071, M and N within the grid (M <= 65535 * 128), out_kind in {bf16, fp16, fp32}.
hipError_t launch_quant_matmul(int out_kind, const void* x, const void* w, const float* sx, const float* sw,
                               const float* bias, int64_t M, int64_t N, int64_t K, void* out, void*,
                               hipStream_t stream) {
  if (M == 0 || N == 0) return hipSuccess;
  QmmArgs a;
  a.x = static_cast<const uint8_t*>(x);
  a.w = static_cast<const uint8_t*>(w);
  a.sx = sx;
  a.sw = sw;
  a.bias = bias;
  a.out = out;
  a.M = (int)M;
  a.N = (int)N;
  a.K = (int)K;
  switch (out_kind) {
    case kQmmBf16: return qmm_launch<kQmmBf16>(a, stream);
    case kQmmFp16: return qmm_launch<kQmmFp16>(a, stream);
    default: return qmm_launch<kQmmFp32>(a, stream);
  }
}

}  // namespace dsa
