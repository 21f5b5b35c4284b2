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
  int* part;          // [splits, M, part_ld] sums of a split product
  int M, N, K, part_ld;
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

// The scaled, biased value of a sum.
__device__ __forceinline__ float qmm_value(const QmmArgs& a, int sum, int n, float sx) {
  float v = (float)sum * sx * a.sw[n];
  if (a.bias) v += a.bias[n];
  return v;
}

// Up to 16 tokens: bound by the weights' bytes.  A workgroup takes 16 output channels and all tokens; its eight
// waves share the rows' bytes, 128 of each row at a time, and load straight into the product's operands, four such
// units ahead (two: 16 tokens of 9216 x 7168 took 23.6 us instead of 21.6; eight: 24.1): nothing is shared between
// waves but the sums, joined through LDS.  Rows may start at any byte; the unit that K ends in is read by chunks that
// are cut there.  One token of 9216 x 7168: 14.2 us, 4.7 TB/s (back to back, 15.5 over weights that no cache holds).
constexpr int kQmmRowWaves = 8;
constexpr int kQmmUnit = 128;
constexpr int kQmmDeep = 4;

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
__global__ __launch_bounds__(kQmmRowWaves * kWave) void qmm_rows_kernel(QmmArgs a) {
  __shared__ __align__(16) int part[kQmmRowWaves][16 * 16];
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const uint8_t* wr = a.w + (int64_t)min(n0 + r, a.N - 1) * a.K;
  const uint8_t* xr = a.x + (int64_t)min(r, a.M - 1) * a.K;

  i32x4 acc = {0, 0, 0, 0};
  u32x4 wv[kQmmDeep][2], xv[kQmmDeep][2];
  auto load = [&](int d, int k) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      __builtin_memcpy(&wv[d][h], wr + k + 64 * h + 16 * g, 16);
      __builtin_memcpy(&xv[d][h], xr + k + 64 * h + 16 * g, 16);
    }
  };
  auto mul = [&](int d) {
#pragma unroll
    for (int h = 0; h < 2; ++h) acc = qmm_mfma(wv[d][h], xv[d][h], acc);
  };
  const int full = a.K / kQmmUnit;  // whole units; wave w takes units w, w + 8, ...
  const int mine = full > wave ? (full - wave + kQmmRowWaves - 1) / kQmmRowWaves : 0;
  const int step = kQmmRowWaves * kQmmUnit;
  int k = wave * kQmmUnit;
#pragma unroll
  for (int d = 0; d < kQmmDeep; ++d)
    if (d < mine) load(d, k + d * step);
  int e = 0;
  for (; e + 2 * kQmmDeep <= mine; e += kQmmDeep) {
#pragma unroll
    for (int d = 0; d < kQmmDeep; ++d) {
      mul(d);
      load(d, k + (kQmmDeep + d) * step);
    }
    k += kQmmDeep * step;
  }
  for (; e < mine; e += kQmmDeep) {  // at most twice
#pragma unroll
    for (int d = 0; d < kQmmDeep; ++d) {
      if (e + d < mine) mul(d);
      if (e + kQmmDeep + d < mine) load(d, k + (kQmmDeep + d) * step);
    }
    k += kQmmDeep * step;
  }
  if (full * kQmmUnit < a.K && full % kQmmRowWaves == wave) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int kk = full * kQmmUnit + 64 * h + 16 * g;
      wv[0][h] = qmm_chunk(wr, kk, a.K);
      xv[0][h] = qmm_chunk(xr, kk, a.K);
    }
    mul(0);
  }
  *reinterpret_cast<i32x4*>(&part[wave][r * 16 + 4 * g]) = acc;
  __syncthreads();
  const int m = tid / 16, n = n0 + tid % 16;
  if (m >= a.M || n >= a.N) return;
  int sum = 0;
#pragma unroll
  for (int v = 0; v < kQmmRowWaves; ++v) sum += part[v][tid];
  qmm_store1<kOut>(a.out, (int64_t)m * a.N + n, qmm_value(a, sum, n, a.sx[m]));
}

// More tokens: kBM x kBN of the output a workgroup, bound by the matrix cores.  The operands' rows stream into
// LDS by DMA, 128 bytes of each at a time, two to four stages; a wave multiplies kTM tokens by 64 channels (32x32x32
// products, channels on the M axis).  Chunk c (16 bytes) of row r lies at c ^ ((r >> 2) & 7), so that the 32 rows
// a half wave reads at one c fall on distinct banks; the DMA fetches the chunks in that order.  Rows start on 16
// bytes and hold whole chunks (qmm_pack_kernel sees to it where they do not); chunks past K come from a row of zeros.
// 16384 x 9216 x 7168: 1042 us (1016 to 1064 by card), 2078 TOP/s; the DMA alone takes 836 us there, the LDS reads 495,
// and the matrix cores reach 3200 to 3700 on random operands (clock); a library 2360 at 8192^3, 2413 at 16384^3.
// With kSplit the steps are dealt to gridDim.z workgroups, which leave int32 sums for qmm_join_kernel.
// Whole lines of a row: with 64 bytes (and four stages) 16384 x 9216 x 7168 took 1120 us, 1089 with 128.
constexpr int kQmmStep = 128;
constexpr int kQmmLanes = kQmmStep / 16;         // of a row in a DMA instruction
constexpr int kQmmRows = kWave / kQmmLanes;      // rows of a DMA instruction
constexpr int kQmmParts = kQmmStep / 32;
__host__ __device__ constexpr int qmm_swz(int row) { return (row / (512 / kQmmStep)) & (kQmmLanes - 1); }
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void qmm_lds_void;
typedef const __attribute__((address_space(1))) void qmm_gbl_void;
static __device__ __align__(128) uint8_t kQmmZeros[16];

// LDS reads as inline asm: through plain loads the compiler would wait for every DMA in flight before each.
template <int kOff>
__device__ __forceinline__ void qmm_b128(u32x4& out, uint32_t addr) {
  __asm__ __volatile__("ds_read_b128 %0, %1 offset:%2" : "=v"(out) : "v"(addr), "i"(kOff));
}
// All but the kLeft youngest LDS reads have returned; v passes through so that no use moves above the wait.
template <int kLeft, int N>
__device__ __forceinline__ void qmm_lds_wait(u32x4 (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) __asm__ __volatile__("" : "+v"(v[i]));
  __asm__ __volatile__("s_waitcnt lgkmcnt(%0)" ::"i"(kLeft) : "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) __asm__ __volatile__("" : "+v"(v[i]));
}

// s_waitcnt with only vmcnt constrained.
template <int N>
__device__ __forceinline__ void qmm_wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}

template <int kBM, int kBN, int kWM, int kWN>
struct QmmShape {
  static constexpr int kWaves = kWM * kWN, kTM = kBM / kWM, kTN = kBN / kWN;
  static constexpr int kFM = kTM / 32, kFN = kTN / 32;
  static constexpr int kStage = (kBM + kBN) * kQmmStep;
  static constexpr int kInstr = (kBM + kBN) / kQmmRows / kWaves;  // DMA instructions of a wave and step
  static_assert((kBM + kBN) % (kQmmRows * kWaves) == 0 && kBN % 32 == 0, "whole DMA instructions");
};

template <int kOut, int kBM, int kBN, int kWM, int kWN, int kStages, bool kSplit>
__global__ __launch_bounds__(kWM* kWN* kWave) void qmm_tile_kernel(QmmArgs a) {
  typedef QmmShape<kBM, kBN, kWM, kWN> S;
  extern __shared__ __align__(16) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  // Consecutive workgroup ids go to the eight XCDs in turn: each XCD takes a run of tiles of its own, in groups of
  // 8 rows of tiles walked column by column, so that the tiles in flight on it share operand rows in its L2.
  const int tm = (a.M + kBM - 1) / kBM, tn = (a.N + kBN - 1) / kBN, tiles = tm * tn;
  int id = blockIdx.x;
  {
    const int per = tiles / 8, rest = tiles % 8, x = id & 7, i = id >> 3;
    id = x * per + min(x, rest) + i;
  }
  constexpr int kGroup = 8;
  const int grp = id / (kGroup * tn), in = id - grp * kGroup * tn;
  const int height = min(kGroup, tm - grp * kGroup);
  const int m0 = (grp * kGroup + in % height) * kBM, n0 = in / height * kBN;
  const int wn = (wave % kWN) * S::kTN, wm = (wave / kWN) * S::kTM;

  const int all = (a.K + kQmmStep - 1) / kQmmStep;
  int s0 = 0, s1 = all;
  if constexpr (kSplit) {
    s0 = (int)((int64_t)all * blockIdx.z / gridDim.z);
    s1 = (int)((int64_t)all * (blockIdx.z + 1) / gridDim.z);
  }
  // The rows of instruction wave + kWaves * j of the stage (channels, then tokens); edge rows repeat the last.
  const uint8_t* src[S::kInstr];
  int chunks[S::kInstr];
#pragma unroll
  for (int j = 0; j < S::kInstr; ++j) {
    const int row = kQmmRows * (wave + S::kWaves * j) + lane / kQmmLanes;
    const bool is_w = row < kBN;
    chunks[j] = 16 * ((lane & (kQmmLanes - 1)) ^ qmm_swz(row));  // kBN is a multiple of 32: the same in either operand
    const int64_t at = is_w ? min(n0 + row, a.N - 1) : min(m0 + row - kBN, a.M - 1);
    src[j] = (is_w ? a.w : a.x) + at * a.K + chunks[j] + (int64_t)s0 * kQmmStep;
  }
  auto dma = [&](int s) {
    uint8_t* dst = lds + s % kStages * S::kStage;
    if ((s + 1) * kQmmStep <= a.K) {
#pragma unroll
      for (int j = 0; j < S::kInstr; ++j) {
        __builtin_amdgcn_global_load_lds((qmm_gbl_void*)src[j], (qmm_lds_void*)(dst + (wave + S::kWaves * j) * 1024), 16,
                                         0, 0);
        src[j] += kQmmStep;
      }
    } else {  // the last step of a K off 128
#pragma unroll
      for (int j = 0; j < S::kInstr; ++j) {
        const uint8_t* p = s * kQmmStep + chunks[j] < a.K ? src[j] : kQmmZeros;
        __builtin_amdgcn_global_load_lds((qmm_gbl_void*)p, (qmm_lds_void*)(dst + (wave + S::kWaves * j) * 1024), 16, 0, 0);
      }
    }
  };
  i32x16 acc[S::kFN][S::kFM];
#pragma unroll
  for (int i = 0; i < S::kFN; ++i)
#pragma unroll
    for (int j = 0; j < S::kFM; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
  const int r = lane & 31, hi = lane >> 5;
  uint32_t off[kQmmParts];
#pragma unroll
  for (int q = 0; q < kQmmParts; ++q) off[q] = r * kQmmStep + 16 * ((2 * q + hi) ^ qmm_swz(r));
  const uint32_t lw = (uint32_t)(uintptr_t)(const qmm_lds_void*)(lds + wn * kQmmStep);
  const uint32_t lx = (uint32_t)(uintptr_t)(const qmm_lds_void*)(lds + (kBN + wm) * kQmmStep);

  // A step's parts (32 bytes of each row): the reads of the next part are in flight under a part's products, across
  // the step's end too, where the barrier lies ahead of the last part's products.
  constexpr int kR = S::kFN + S::kFM;
  u32x4 v[2][kR];
  auto read = [&](u32x4(&o)[kR], int s, int q) {
    const uint32_t st = s % kStages * S::kStage, w = lw + st + off[q], x = lx + st + off[q];
    qmm_b128<0>(o[0], w);
    qmm_b128<32 * kQmmStep>(o[1], w);
    qmm_b128<0>(o[2], x);
    if constexpr (S::kFM > 1) qmm_b128<32 * kQmmStep>(o[3], x);
    if constexpr (S::kFM > 2) qmm_b128<64 * kQmmStep>(o[4], x);
    if constexpr (S::kFM > 3) qmm_b128<96 * kQmmStep>(o[5], x);
  };
  static_assert(S::kFN == 2 && S::kFM <= 4, "the reads above");
  auto mul = [&](const u32x4(&o)[kR]) {
#pragma unroll
    for (int j = 0; j < S::kFM; ++j)
#pragma unroll
      for (int i = 0; i < S::kFN; ++i)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, o[i]),
                                                          __builtin_bit_cast(i32x4, o[S::kFN + j]), acc[i][j], 0, 0, 0);
  };
  // This wave's part of step s is in LDS (up to kStages - 2 younger steps may be in flight); behind the barrier
  // everyone's is, and all reads of the step before it are done.
  auto turn = [&](int s) {
    const int younger = min(kStages - 2, s1 - 1 - s);
    if (kStages > 3 && younger == 2) qmm_wait_vmcnt<2 * S::kInstr>();
    else if (kStages > 2 && younger == 1) qmm_wait_vmcnt<S::kInstr>();
    else qmm_wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i)
    if (s0 + i < s1) dma(s0 + i);
  turn(s0);
  if (s0 + kStages - 1 < s1) dma(s0 + kStages - 1);
  read(v[0], s0, 0);
  auto parts = [&](int s) {  // all products of the stage but the last part's, whose operands are left in v[1]
#pragma unroll
    for (int q = 0; q < kQmmParts - 1; ++q) {
      read(v[(q + 1) & 1], s, q + 1);
      qmm_lds_wait<kR>(v[q & 1]);
      mul(v[q & 1]);
    }
    qmm_lds_wait<0>(v[1]);
  };
  for (int s = s0; s + 1 < s1; ++s) {
    parts(s);
    turn(s + 1);
    if (s + kStages < s1) dma(s + kStages);
    read(v[0], s + 1, 0);
    mul(v[1]);
  }
  parts(s1 - 1);
  mul(v[1]);

  // Lane (r, hi) holds channels 8 c + 4 hi + e (c = 0 .. 3, e = 0 .. 3) of token r of a 32 x 32 block.
  // A wave turns 32 rows of the output at a time in its own LDS and stores neighbouring channels from neighbouring
  // lanes, wherever rows start.  Straight from the sums' places, four channels or one a lane: 16384 x 9216 x 7168 takes
  // 1085 us instead of 1051, 16384 x 9215 x 7168 1306 instead of 1062, and with the sums of split products 1021 x 2113 x
  // 4099 34.9 instead of 33.4.
  constexpr int kLd = S::kTN + 4;  // 16 lanes' writes of 16 bytes meet each bank once
  static_assert(S::kTN == kWave && S::kWaves * 32 * kLd * 4 <= kStages * S::kStage, "a channel a lane, in the stages");
  __syncthreads();  // no wave reads its operands any more
  int* turned = reinterpret_cast<int*>(lds) + wave * 32 * kLd;
  const int n = n0 + wn + lane;
#pragma unroll
  for (int j = 0; j < S::kFM; ++j) {
    const int m1 = m0 + wm + 32 * j;
#pragma unroll
    for (int i = 0; i < S::kFN; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<i32x4*>(turned + r * kLd + 32 * i + 8 * c + 4 * hi) =
            i32x4{acc[i][j][4 * c], acc[i][j][4 * c + 1], acc[i][j][4 * c + 2], acc[i][j][4 * c + 3]};
    // A wave's LDS accesses keep their order.
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (n < a.N) {
#pragma unroll 4
      for (int t = 0; t < min(32, a.M - m1); ++t) {
        const int sum = turned[t * kLd + lane];
        if constexpr (kSplit) a.part[((int64_t)blockIdx.z * a.M + m1 + t) * a.part_ld + n] = sum;
        else qmm_store1<kOut>(a.out, (int64_t)(m1 + t) * a.N + n, qmm_value(a, sum, n, a.sx[m1 + t]));
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// Sums of the splits, scaled and biased: four channels a thread where rows of the output start on them, otherwise four
// elements 256 apart (neighbouring lanes then store neighbouring elements).  Split products have at most 170 tiles, so
// elements are counted in 32 bits.
template <int kOut, bool kQuad>
__global__ __launch_bounds__(256) void qmm_join_kernel(QmmArgs a, int splits) {
  const uint32_t per_row = kQuad ? a.part_ld / 4 : a.N, all = (uint32_t)a.M * per_row;
  const int64_t step = (int64_t)a.M * a.part_ld;
  if constexpr (kQuad) {
    const uint32_t t = blockIdx.x * 256 + threadIdx.x;
    if (t >= all) return;
    const uint32_t m = t / per_row, n = 4 * (t - m * per_row);
    const int* from = a.part + (int64_t)m * a.part_ld + n;
    const float sx = a.sx[m];
    i32x4 sum = {0, 0, 0, 0};
#pragma unroll 2
    for (int z = 0; z < splits; ++z) sum += *reinterpret_cast<const i32x4*>(from + z * step);
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = qmm_value(a, sum[e], n + e, sx);
    qmm_store4<kOut>(a.out, (int64_t)m * a.N + n, v);
  } else {
    const uint32_t t0 = blockIdx.x * 1024 + threadIdx.x;
    uint32_t m[4], n[4];
    int sum[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t t = min(t0 + 256 * e, all - 1);
      m[e] = t / per_row;
      n[e] = t - m[e] * per_row;
    }
    for (int z = 0; z < splits; ++z)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += a.part[z * step + (int64_t)m[e] * a.part_ld + n[e]];
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = qmm_value(a, sum[e], n[e], a.sx[m[e]]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (t0 + 256 * e < all) qmm_store1<kOut>(a.out, (int64_t)(t0 + 256 * e), v[e]);
  }
}

// Rows of K bytes anywhere to rows of ld bytes (a multiple of 128) on 16 bytes, zeros behind K: a wave a row.
__global__ __launch_bounds__(256) void qmm_pack_kernel(const uint8_t* x, int64_t M, const uint8_t* w, int64_t N, int K,
                                                       int ld, uint8_t* to) {
  const int64_t row = (int64_t)blockIdx.x * (256 / kWave) + threadIdx.x / kWave;
  if (row >= M + N) return;
  const uint8_t* src = row < M ? x + row * K : w + (row - M) * K;
  uint8_t* dst = to + row * ld;
#pragma unroll 4
  for (int k = 16 * (threadIdx.x & (kWave - 1)); k < ld; k += 16 * kWave)
    *reinterpret_cast<u32x4*>(dst + k) = qmm_chunk(src, k, K);
}

// The launch of a call: which kernel, and the workspace's parts.
struct QmmPlan {
  int tile;    // 16: the kernel for few tokens; 32, 64, 128: tokens of a tile of 128 channels; 256: of 256 channels
  bool pack;   // operands copied to aligned rows first
  int splits;  // workgroups that share a tile's K
  bool deep;   // tiles of 128 with four stages, one workgroup a CU
  size_t pack_bytes, part_bytes;
};

static int64_t qmm_ld(int64_t K) { return (K + 127) / 128 * 128; }

// `odd`: rows do not start on 16 bytes or hold no whole number of chunks.
static QmmPlan qmm_plan(int64_t M, int64_t N, int64_t K, bool odd) {
  QmmPlan p = {16, false, 1, false, 0, 0};
  // Up to 16 tokens every workgroup reads all of x beside its 16 rows of w.  Rows and (shared) tiles, us: one token of
  // 9216 x 7168 15.5 and 19.2, of 4096 x 4096 5.7 and 9.5; 16 tokens of 4096 x 7168 8.5 and 12.0, of 8192 x 4096 9.8 and
  // 11.8, but of 9216 x 7168 21.8 and 20.1, of 7168 x 8192 18.4 and 16.1: from 12 tokens on tiles are up to 3 us ahead
  // where the weights come from memory, as much behind where a cache holds them.  Past 16 this kernel has no form.
  if (M <= 16) return p;
  p.pack = odd;
  if (odd) p.pack_bytes = (size_t)((M + N) * qmm_ld(K));
  p.tile = M <= 32 ? 32 : M <= 64 ? 64 : 128;
  const int64_t small = ((M + p.tile - 1) / p.tile) * ((N + 127) / 128);
  const int64_t big = ((M + 255) / 256) * ((N + 255) / 256);
  // The larger tile multiplies 1.2 times as fast (8192^3: 1932 against 1595 TOP/s); a round of 256 of them takes what
  // two rounds of 512 of the smaller one would at one speed.  Rounds count the rows past M that a tile multiplies too.
  // Smaller and larger tile, us: with K = 4096, 128 x 32768 41 and 69, 128 x 131072 148 and 172, 300 x 32768 87 and 77,
  // 300 x 131072 298 and 304, 520 x 32768 128 and 137, 6144 x 6144 196 and 208 (the one of these that the rule misses);
  // with K = 7168, 1100 x 9216 126 and 107, 2100 x 9216 193 and 209, 4096 x 9216 372 and 342.
  const int64_t rounds_big = (big + 255) / 256, rounds_small = (small + 511) / 512;
  if (p.tile == 128 && 0.82 * 2 * (double)rounds_big < (double)rounds_small) {
    p.tile = 256;
    return p;
  }
  // Few tiles share their K, eight steps each at least, up to about one workgroup a CU: with up to two, what the
  // join reads costs more (64 tokens of 7168 x 8192: 22.0 us instead of 18.0; 512: 57.2 instead of 51).  More than
  // half as many tiles of 128 as CUs, and at most 170, whose three shares fill two workgroups a CU, share a long K by
  // three.  Aligned rows, us with one share and with three, by steps of K:
  //   tiles                20          32          33          36          40          56          72
  //   136 (1024 x 2112)    21.1 24.8   28.0 27.3   30.3 27.7   29.4 27.1   33.5 29.6   41.0 35.1   52.0 39.5
  //   154 (1408 x 1792)    22.2 25.8   28.7 30.2   28.3 27.7   29.5 28.3   34.4 31.7   41.8 37.3   52.5 43.0
  //   169 (1664 x 1664)    22.4 27.6   29.2 31.4   28.2 28.6   29.7 29.5   35.0 32.9   42.8 38.6   53.7 44.6
  //   170 (256 x 10880)    22.3 30.1   30.4 34.3   30.4 32.1   32.0 33.2   37.9 39.5   45.0 44.4   55.9 51.4
  // so the sides cross between 31 steps (fewest tiles) and 38 (most); the wide product of two rows of tiles, bound by its
  // weights, crosses at 56.  Copied rows gain from about 20 steps on but for such wide ones (136 tiles, 27 steps: 33.5 and
  // 30.5; 169: 34.8 and 33.0; 170, 256 x 10880: 44.5 and 47.2); they keep to the same bound.
  const int64_t steps = (K + kQmmStep - 1) / kQmmStep;
  if (p.tile == 128 && small > 128 && small <= 170 && steps > 32) p.splits = 3;
  else
    while (p.splits < 8 && small * p.splits * 2 <= 256 && steps >= 8 * p.splits) p.splits *= 2;
  // A workgroup alone on its CU keeps three steps in flight (512 tokens: 65.0 -> 52 us).
  p.deep = p.tile == 128 && small * p.splits <= 256;
  if (p.splits > 1) p.part_bytes = (size_t)(p.splits * M * ((N + 3) / 4 * 4) * 4);
  return p;
}

static bool qmm_odd_rows(const void* x, const void* w, int64_t K) {
  return K % 16 != 0 || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) != 0;
}

// The largest grid within the 2^32 threads of a launch: 16 channels or a tile a workgroup, the copies a row a wave (a
// join's is smaller than its tiles').
bool quant_matmul_fits(int64_t M, int64_t N, int64_t K, bool aligned) {
  const QmmPlan p = qmm_plan(M, N, K, !aligned || K % 16 != 0);
  const int64_t most = ((int64_t)1 << 32) - 1024;
  if (p.tile == 16) return (N + 15) / 16 * kQmmRowWaves * kWave <= most;
  if (p.pack && (M + N) * kWave > most) return false;
  const int64_t bm = p.tile, bn = p.tile == 256 ? 256 : 128, threads = p.tile == 256 ? 512 : p.tile == 32 ? 128 : 256;
  return ((M + bm - 1) / bm) * ((N + bn - 1) / bn) * threads <= most;
}

// `aligned`: the operands start on 16 bytes.
size_t quant_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K, bool aligned) {
  const QmmPlan p = qmm_plan(M, N, K, !aligned || K % 16 != 0);
  return p.pack_bytes + p.part_bytes;
}

template <int kOut, int kBM, int kBN, int kWM, int kWN, int kStages, bool kSplit>
static hipError_t qmm_launch_tile(const QmmArgs& a, int splits, hipStream_t stream) {
  constexpr int lds = kStages * QmmShape<kBM, kBN, kWM, kWN>::kStage;
  static_assert(kStages >= 2 && kStages <= 4 && lds <= 160 * 1024, "LDS");
  const hipError_t e = set_dynamic_lds_once<qmm_tile_kernel<kOut, kBM, kBN, kWM, kWN, kStages, kSplit>>(lds);
  if (e != hipSuccess) return e;
  const dim3 grid((unsigned)(((a.M + kBM - 1) / kBM) * ((a.N + kBN - 1) / kBN)), 1, splits);
  hipLaunchKernelGGL((qmm_tile_kernel<kOut, kBM, kBN, kWM, kWN, kStages, kSplit>), grid, dim3(kWM * kWN * kWave), lds,
                     stream, a);
  return hipGetLastError();
}

template <int kOut, int kBM, int kWM, int kWN, int kStages>
static hipError_t qmm_launch_shared(const QmmArgs& a, int splits, hipStream_t stream) {
  if (splits == 1) return qmm_launch_tile<kOut, kBM, 128, kWM, kWN, kStages, false>(a, 1, stream);
  const hipError_t e = qmm_launch_tile<kOut, kBM, 128, kWM, kWN, kStages, true>(a, splits, stream);
  if (e != hipSuccess) return e;
  if ((a.N & 3) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0) {
    const int64_t quads = (int64_t)a.M * (a.part_ld / 4);
    hipLaunchKernelGGL((qmm_join_kernel<kOut, true>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, stream, a, splits);
  } else {
    const int64_t all = (int64_t)a.M * a.N;
    hipLaunchKernelGGL((qmm_join_kernel<kOut, false>), dim3((unsigned)((all + 1023) / 1024)), dim3(256), 0, stream, a, splits);
  }
  return hipGetLastError();
}

template <int kOut>
static hipError_t qmm_launch(QmmArgs a, void* workspace, hipStream_t stream) {
  const QmmPlan p = qmm_plan(a.M, a.N, a.K, qmm_odd_rows(a.x, a.w, a.K));
  if (p.tile == 16) {
    hipLaunchKernelGGL((qmm_rows_kernel<kOut>), dim3((unsigned)((a.N + 15) / 16)), dim3(kQmmRowWaves * kWave), 0, stream,
                       a);
    return hipGetLastError();
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.part = reinterpret_cast<int*>(ws + p.pack_bytes);
  a.part_ld = (a.N + 3) / 4 * 4;
  if (p.pack) {
    const int ld = (int)qmm_ld(a.K);
    hipLaunchKernelGGL(qmm_pack_kernel, dim3((unsigned)(((int64_t)a.M + a.N + 3) / 4)), dim3(256), 0, stream, a.x,
                       (int64_t)a.M, a.w, (int64_t)a.N, a.K, ld, ws);
    a.x = ws;
    a.w = ws + (int64_t)a.M * ld;
    a.K = ld;
  }
  switch (p.tile) {
    case 32: return qmm_launch_shared<kOut, 32, 1, 2, 3>(a, p.splits, stream);
    case 64: return qmm_launch_shared<kOut, 64, 2, 2, 3>(a, p.splits, stream);
    case 128:
      if (p.deep) return qmm_launch_shared<kOut, 128, 2, 2, 4>(a, p.splits, stream);
      return qmm_launch_shared<kOut, 128, 2, 2, 2>(a, p.splits, stream);
    default: return qmm_launch_tile<kOut, 256, 256, 2, 4, 2, false>(a, 1, stream);
  }
}

// Caller validated: 1 <= K <= 131071, quant_matmul_fits, out_kind in {bf16, fp16, fp32}, a workspace of
// quant_matmul_workspace_bytes.
hipError_t launch_quant_matmul(int out_kind, const void* x, const void* w, const float* sx, const float* sw,
                               const float* bias, int64_t M, int64_t N, int64_t K, void* out, void* workspace,
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
  a.part = nullptr;
  a.part_ld = 0;
  switch (out_kind) {
    case kQmmBf16: return qmm_launch<kQmmBf16>(a, workspace, stream);
    case kQmmFp16: return qmm_launch<kQmmFp16>(a, workspace, stream);
    default: return qmm_launch<kQmmFp32>(a, workspace, stream);
  }
}

}  // namespace dsa
