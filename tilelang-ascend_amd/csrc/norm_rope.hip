// Norms of queries and keys for each head with the position rotation in the same pass; keys and values go to the
// rows of a paged cache in the same launch where one is given.
//
//   y = x / sqrt(mean_j x_j^2 + eps) * w                        (each head's D elements, fp32)
//   (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)                 for the pairs of the first R elements,
//
// c, s = cos / sin[position of the token, pair]; pair i is (i, i + R/2), or (2i, 2i + 1) with interleaved; the
// other elements keep y.  One rounding, to the output type.  HBM bound: each element read and written once.
//
// A head's row is held by a group of kL lanes, 8 elements (16 bytes) a lane, as many lanes as the row has chunks
// (rounded up to a power of two), so a 256-byte row takes 16 lanes and a wave works on four rows.  The partner of
// an element of the first form lies R/2 elements away: R/16 lanes, one shuffle an element.
#include "common.hpp"

namespace dsa {

struct NormRopeArgs {
  const uint16_t *q, *k, *v;  // token t's heads at q + t * q_stride, D elements each
  int64_t q_stride, k_stride, v_stride;
  const void *qw, *kw;  // [D], 16-bit or fp32, or null (ones)
  const int32_t* positions;
  const float *cos, *sin;  // [table, R / 2]
  const int32_t* slots;    // null: keys go to k_out
  uint16_t *q_out, *k_out;  // [T, H, D], [T, G, D] or the caches [rows, G, D]
  uint16_t* v_out;
  int T, H, G, D, R, table, w_f32;
  int64_t rows;  // of the caches
  float eps;
};

template <bool kF16>
__device__ __forceinline__ float nr_get(uint32_t w, int hi) {
  const uint16_t u = (uint16_t)(hi ? w >> 16 : w);
  if constexpr (kF16) return (float)__builtin_bit_cast(_Float16, u);
  else return __uint_as_float((uint32_t)u << 16);
}

template <bool kF16>
__device__ __forceinline__ uint32_t nr_pack(float lo, float hi) {
  if constexpr (kF16) {
    const _Float16 a = (_Float16)lo, b = (_Float16)hi;
    return (uint32_t)__builtin_bit_cast(uint16_t, a) | ((uint32_t)__builtin_bit_cast(uint16_t, b) << 16);
  } else {
    return pack_bf16x2(lo, hi);
  }
}

// Row n of a token's H + G (+ G) rows: a query head, a key head or, with a cache, a value head.
template <bool kF16, int kL, bool kPairs>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeArgs a) {
  const int l = threadIdx.x & (kL - 1);
  const int heads = a.H + a.G + (a.slots ? a.G : 0);
  const int64_t row = (int64_t)blockIdx.x * (256 / kL) + threadIdx.x / kL;
  // A group past the last row repeats it and stores nothing: its lanes take part in the shuffles.
  const int64_t last = (int64_t)a.T * heads - 1;
  const int64_t rr = row < last ? row : last;
  const int t = (int)(rr / heads), n = (int)(rr - (int64_t)t * heads);
  const bool is_q = n < a.H, is_v = n >= a.H + a.G;
  const int h = is_q ? n : is_v ? n - a.H - a.G : n - a.H;
  const bool in = 8 * l < a.D;
  const uint16_t* src = (is_q ? a.q + t * a.q_stride : is_v ? a.v + t * a.v_stride : a.k + t * a.k_stride) +
                        (int64_t)h * a.D + (in ? 8 * l : 0);
  const u32x4 x = *reinterpret_cast<const u32x4*>(src);
  const int pos = a.positions[t];
  const bool pos_ok = pos >= 0 && pos < a.table;

  // The destination: outputs are rows of all tokens, caches rows of the slots that lie in them.
  uint16_t* dst = nullptr;
  if (is_q) {
    dst = a.q_out + ((int64_t)t * a.H + h) * a.D;
  } else if (a.slots) {
    const int64_t slot = a.slots[t];
    if (slot >= 0 && slot < a.rows && pos_ok) dst = (is_v ? a.v_out : a.k_out) + (slot * a.G + h) * a.D;
  } else {
    dst = a.k_out + ((int64_t)t * a.G + h) * a.D;
  }
  const bool store = in && row <= last && dst != nullptr;

  float y[8];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = nr_get<kF16>(x[i / 2], i & 1);
    sum += in ? y[i] * y[i] : 0.f;
  }
#pragma unroll
  for (int o = kL / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
  const float inv = 1.f / sqrtf(sum / (float)a.D + a.eps);
  const void* w = is_q ? a.qw : a.kw;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float wi = 1.f;
    if (w && in) {
      if (a.w_f32) {
        wi = static_cast<const float*>(w)[8 * l + i];
      } else {
        const uint16_t u = static_cast<const uint16_t*>(w)[8 * l + i];
        wi = nr_get<kF16>(u, 0);
      }
    }
    y[i] = y[i] * inv * wi;
  }
  const int half = a.R / 2;
  const bool rot = 8 * l < a.R;
  const int64_t tab = (int64_t)(pos_ok ? pos : 0) * half;
  if constexpr (kPairs) {
    if (rot) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float c = a.cos[tab + 4 * l + i], s = a.sin[tab + 4 * l + i];
        const float ya = y[2 * i], yb = y[2 * i + 1];
        y[2 * i] = ya * c - yb * s;
        y[2 * i + 1] = yb * c + ya * s;
      }
    }
  } else {
    // Lanes below R/16 hold the first elements of the pairs, the next R/16 the second ones.
    const int d = a.R / 16;
    const bool second = l >= d;
    const int lane = threadIdx.x & (kWave - 1);
    const int other = second ? lane - d : lane + d;
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __shfl(y[i], rot ? other : lane, kWave);
    if (rot) {
      const int at = 8 * (second ? l - d : l);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float c = a.cos[tab + at + i], s = a.sin[tab + at + i];
        y[i] = second ? y[i] * c + p[i] * s : y[i] * c - p[i] * s;
      }
    }
  }
  if (!store) return;
  u32x4 o;
  if (is_v) {
    o = x;
  } else if (!pos_ok) {
    o = u32x4{0, 0, 0, 0};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = nr_pack<kF16>(y[2 * i], y[2 * i + 1]);
  }
  *reinterpret_cast<u32x4*>(dst + 8 * l) = o;
}

template <bool kF16, int kL>
static hipError_t nr_launch(const NormRopeArgs& a, bool pairs, hipStream_t stream) {
  const int64_t rows = (int64_t)a.T * (a.H + a.G + (a.slots ? a.G : 0));
  const dim3 grid((unsigned)((rows + 256 / kL - 1) / (256 / kL)));
  if (pairs)
    hipLaunchKernelGGL((norm_rope_kernel<kF16, kL, true>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((norm_rope_kernel<kF16, kL, false>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

// Caller validated: D a multiple of 8 in [8, 512], R a multiple of 16 in [0, D], strides multiples of 8, 16-byte
// aligned pointers, T * (H + 2 G) * 8 < 2^31 * 256 / 64.
template <bool kF16>
static hipError_t nr_dispatch(const NormRopeArgs& a, bool pairs, hipStream_t stream) {
  const int chunks = a.D / 8;
  if (chunks <= 8) return nr_launch<kF16, 8>(a, pairs, stream);
  if (chunks <= 16) return nr_launch<kF16, 16>(a, pairs, stream);
  if (chunks <= 32) return nr_launch<kF16, 32>(a, pairs, stream);
  return nr_launch<kF16, 64>(a, pairs, stream);
}

hipError_t launch_qk_norm_rope(int is_fp16, const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                               const void* v, int64_t v_stride, const void* qw, const void* kw, int w_f32,
                               const int32_t* positions, const float* cos, const float* sin, int64_t table,
                               int64_t T, int64_t H, int64_t G, int64_t D, int64_t R, float eps, int interleaved,
                               const int32_t* slots, int64_t rows, void* q_out, void* k_out, void* v_out,
                               hipStream_t stream) {
  if (T == 0 || H + G == 0) return hipSuccess;
  NormRopeArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.qw = qw;
  a.kw = kw;
  a.positions = positions;
  a.cos = cos;
  a.sin = sin;
  a.slots = slots;
  a.q_out = static_cast<uint16_t*>(q_out);
  a.k_out = static_cast<uint16_t*>(k_out);
  a.v_out = static_cast<uint16_t*>(v_out);
  a.T = (int)T;
  a.H = (int)H;
  a.G = (int)G;
  a.D = (int)D;
  a.R = (int)R;
  a.table = (int)table;
  a.w_f32 = w_f32;
  a.rows = rows;
  a.eps = eps;
  return is_fp16 ? nr_dispatch<true>(a, interleaved, stream) : nr_dispatch<false>(a, interleaved, stream);
}

}  // namespace dsa
