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
// (rounded up to a power of two), so a 256-byte row takes 16 lanes and a wave works on four tokens' rows at once.  A
// group takes kRows heads of one token, whose loads all go out before the first is used and which share the token's
// angles (32768 tokens of 72 rows of 128: 492 us with a head a group, 222 with four, 5.5 TB/s).  The partner of an
// element of the first form lies R/2 elements away: R/16 lanes, one shuffle an element.
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
  int T, H, G, D, R, table, w_f32, heads;  // heads: rows of a token, H + G (+ G with a cache)
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

// Eight weights of chunk l: fp32, 16 bits, or ones.
template <bool kF16>
__device__ __forceinline__ void nr_weights(float (&w)[8], const void* p, int f32, int l) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (!p) return;
  if (f32) {
    __builtin_memcpy(w, static_cast<const float*>(p) + 8 * l, 32);
  } else {
    u32x4 v;
    __builtin_memcpy(&v, static_cast<const uint16_t*>(p) + 8 * l, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = nr_get<kF16>(v[i / 2], i & 1);
  }
}

// Row n of a token's `heads` rows: a query head, a key head or, with a cache, a value head.
template <bool kF16, int kL, bool kPairs, int kRows>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeArgs a) {
  const int l = threadIdx.x & (kL - 1);
  const uint32_t sets = (uint32_t)(a.heads + kRows - 1) / kRows;  // of a token
  // A group past the last set repeats it and stores nothing: its lanes take part in the shuffles.
  const uint32_t all = (uint32_t)a.T * sets, mine = blockIdx.x * (256 / kL) + threadIdx.x / kL;
  const uint32_t set = mine < all ? mine : all - 1;
  const int t = (int)(set / sets), n0 = (int)(set - (uint32_t)t * sets) * kRows;
  const bool in = 8 * l < a.D;
  const int lc = in ? l : 0;
  const int pos = a.positions[t];
  const bool pos_ok = pos >= 0 && pos < a.table;
  const int64_t slot = a.slots ? a.slots[t] : -1;

  u32x4 x[kRows];
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int n = min(n0 + j, a.heads - 1);
    const uint16_t* src = n < a.H         ? a.q + t * a.q_stride + (int64_t)n * a.D
                          : n < a.H + a.G ? a.k + t * a.k_stride + (int64_t)(n - a.H) * a.D
                                          : a.v + t * a.v_stride + (int64_t)(n - a.H - a.G) * a.D;
    x[j] = *reinterpret_cast<const u32x4*>(src + 8 * lc);
  }
  float qw[8], kw[8];
  nr_weights<kF16>(qw, a.qw, a.w_f32, lc);
  nr_weights<kF16>(kw, a.kw, a.w_f32, lc);
  // The angles of this lane's pairs: four with interleaved elements, eight otherwise (lanes below R/16 hold the first
  // elements of the pairs, the next R/16 the second ones).
  constexpr int kA = kPairs ? 4 : 8;
  const int half = a.R / 2, d = a.R / 16;
  const bool rot = 8 * l < a.R, second = !kPairs && l >= d;
  const int64_t tab = (int64_t)(pos_ok && rot ? pos : 0) * half + (rot ? kA * (second ? l - d : l) : 0);
  float c[kA], sn[kA];
  if (a.R > 0 && a.table > 0) {
    __builtin_memcpy(c, a.cos + tab, sizeof(c));
    __builtin_memcpy(sn, a.sin + tab, sizeof(sn));
  }
  const int lane = threadIdx.x & (kWave - 1);
  const int other = !rot ? lane : second ? lane - d : lane + d;

#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int n = n0 + j;
    float y[8], sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = nr_get<kF16>(x[j][i / 2], i & 1);
      sum += in ? y[i] * y[i] : 0.f;
    }
#pragma unroll
    for (int o = kL / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
    const float inv = 1.f / sqrtf(sum / (float)a.D + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = y[i] * inv * (n < a.H ? qw[i] : kw[i]);
    if constexpr (kPairs) {
      if (rot) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float ya = y[2 * i], yb = y[2 * i + 1];
          y[2 * i] = ya * c[i] - yb * sn[i];
          y[2 * i + 1] = yb * c[i] + ya * sn[i];
        }
      }
    } else {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = __shfl(y[i], other, kWave);
      if (rot) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = second ? y[i] * c[i] + p[i] * sn[i] : y[i] * c[i] - p[i] * sn[i];
      }
    }
    // The destination: outputs are rows of all tokens, caches rows of the slots that lie in them.
    uint16_t* dst = nullptr;
    if (n < a.H) {
      dst = a.q_out + ((int64_t)t * a.H + n) * a.D;
    } else if (a.slots) {
      const int h = n < a.H + a.G ? n - a.H : n - a.H - a.G;
      if (slot >= 0 && slot < a.rows && pos_ok) dst = (n < a.H + a.G ? a.k_out : a.v_out) + (slot * a.G + h) * a.D;
    } else {
      dst = a.k_out + ((int64_t)t * a.G + n - a.H) * a.D;
    }
    if (!in || mine >= all || n >= a.heads || !dst) continue;
    u32x4 o;
    if (n >= a.H + a.G) {
      o = x[j];
    } else if (!pos_ok) {
      o = u32x4{0, 0, 0, 0};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = nr_pack<kF16>(y[2 * i], y[2 * i + 1]);
    }
    *reinterpret_cast<u32x4*>(dst + 8 * l) = o;
  }
}

template <bool kF16, int kL, bool kPairs, int kRows>
static void nr_launch_rows(const NormRopeArgs& a, hipStream_t stream) {
  const int64_t sets = (int64_t)a.T * ((a.heads + kRows - 1) / kRows);
  const dim3 grid((unsigned)((sets + 256 / kL - 1) / (256 / kL)));
  hipLaunchKernelGGL((norm_rope_kernel<kF16, kL, kPairs, kRows>), grid, dim3(256), 0, stream, a);
}

// Four heads a group where 2048 workgroups are left, one otherwise.
static bool nr_many(int64_t T, int64_t heads, int lanes) { return T * heads * lanes >= (int64_t)2048 * 256 * 4; }

// The grid lies within the 2^32 threads of a launch; `heads`: rows of a token.
bool qk_norm_rope_fits(int64_t T, int64_t heads, int64_t D) {
  const int lanes = D <= 64 ? 8 : D <= 128 ? 16 : D <= 256 ? 32 : 64;
  const int64_t sets = T * (nr_many(T, heads, lanes) ? (heads + 3) / 4 : heads);
  return sets * lanes <= ((int64_t)1 << 32) - 512;
}

template <bool kF16, int kL>
static hipError_t nr_launch(const NormRopeArgs& a, bool pairs, hipStream_t stream) {
  const bool many = nr_many(a.T, a.heads, kL);
  if (pairs) many ? nr_launch_rows<kF16, kL, true, 4>(a, stream) : nr_launch_rows<kF16, kL, true, 1>(a, stream);
  else many ? nr_launch_rows<kF16, kL, false, 4>(a, stream) : nr_launch_rows<kF16, kL, false, 1>(a, stream);
  return hipGetLastError();
}

// Caller validated: D a multiple of 8 in [8, 512], R a multiple of 16 in [0, D], strides multiples of 8, 16-byte
// aligned pointers, T * (H + 2 G) < 2^31, qk_norm_rope_fits.
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
  a.heads = (int)(H + G + (slots ? G : 0));
  a.rows = rows;
  a.eps = eps;
  return is_fp16 ? nr_dispatch<true>(a, interleaved, stream) : nr_dispatch<false>(a, interleaved, stream);
}

}  // namespace dsa
