// Attention of new tokens over a paged cache: grouped heads, 64 or 128 wide, gfx950.
//
// Sequence b brings S_b query tokens, the last S_b of its n_b keys; its keys and values lie in pages of two pools
// [blocks, block_size, G, D], key j in row table[b, j / block_size] * block_size + j % block_size.  Query heads
// g * Hg .. (g + 1) * Hg - 1 (Hg = H / G) read KV head g:
//   score_j   = sm_scale * q[t, h, :] . k[j, g, :]           over the keys that the token sees
//   out[t, h] = sum_j exp(score_j - lse) v[j, g, :],  lse = ln(sum_j exp(score_j) + exp(sink_h))
// Token i of S_b sits at position p = n_b - S_b + i and sees key j iff 0 <= j < n_b, j <= p (causal),
// j >= p - win_left (with a window), and the key's page lies in the pool.  A row that sees nothing gives 0, and
// lse = -inf (or its sink).
//
// Rows.  The Hg heads of a group's tokens are rows of one product: row rho = i * Hg + h of sequence b and group g,
// cut into tiles of kR rows, so that each key is read once for a tile whatever Hg.  Tile i of sequence b has
// the slot floor(start_b * Hg / kR) + b + i: sequences get disjoint slots without a prefix sum, and a grid of
// floor(T * Hg / kR) + B + 1 slots holds them all (b = B is the padding behind the last packed sequence).
//
// Two ways over a tile's keys, by rows per sequence (pg_plan):
//  - pg_keys: 16 or 32 rows, for decode batches, bound by the caches' bytes.  Four waves hold the same rows and
//    take 32 keys each of a unit of 128, every wave with a ring of its own in LDS and no barrier in the loop; the
//    waves' sums are merged at the end.
//  - pg_rows: 256 rows, 32 a wave, for chunks and prompts, bound by matrix cores, exponentials and LDS reads alike.
//    Eight waves share tiles of 64 keys in LDS.  Waves w and w + 4 lie on one SIMD and take turns: one
//    multiplies (scores of a tile and the products of the tile before with V) while the other takes exponentials.
//
// Work split.  Where there are tiles enough a workgroup takes a tile and all its keys.  Otherwise the units of all
// tiles form one line that is cut into equal parts, a workgroup each, so that batches of uneven lengths load
// the card evenly; a tile whose line is cut leaves parts (unnormalised sums in fp32, with maximum and sum) that a
// second launch joins.
//
// S^T = K Q^T with keys on the M axis, so that a lane holds many scores of one row; softmax in base 2; O^T += V^T P^T
// with V^T through transposing LDS reads.  Probabilities are rounded to the caches' 16 bits for that product, whose matrix
// instructions take them so (bf16 outputs: 0.0019 to 0.0024 off where an fp32 form rounded once has 0.0015 to 0.0017); the
// sum of them is taken before the rounding, in fp32, as maxima and all sums are.
#include <type_traits>

#include "gqa_common.hpp"

namespace dsa {

constexpr int kPgTile = 32;                 // keys a wave of pg_keys takes at once
constexpr int kPgWaves = 4;
constexpr int kPgThreads = kPgWaves * kWave;
constexpr int kPgUnit = kPgWaves * kPgTile;  // 128 keys
constexpr int kPgMaxSlots = 4096;            // of a call whose tiles share the line of units
constexpr int kPgFewSlots = 256;             // of all groups: the join takes a pass a workgroup
constexpr float kPgInf = __builtin_huge_valf();

struct PgArgs {
  const uint16_t* q;   // [T, H, D]
  const uint16_t* kc;  // [rows, G, D]
  const uint16_t* vc;
  const int32_t* table;   // [B, max_blocks]
  const int32_t* cu_q;    // [B] inclusive prefix sums, or null: sequence b has rows b * S ..
  const int32_t* q_len;   // [B] or null (S); with cu_q unused
  const int32_t* kv_len;  // [B]
  const float* sinks;     // [H] or null
  uint16_t* out;          // [T, H, D]
  float* lse;             // [T, H]
  float* part;            // parts: sums [kR, D], then (maximum, sum) [kR, 2]
  int32_t* line;          // [slots + 1] the line's `at`, then [slots] its `seq`, for the join
  int T, B, S, H, G, Hg, block_size, max_blocks, num_blocks, causal, win, wgs;
  int slots;              // of the call
  uint32_t div_mul;       // j / block_size = umulhi(j, div_mul) >> div_shift for 0 <= j < 2^31; 0: block_size is 1
  int div_shift;
  float scale_log2;  // sm_scale * log2(e)
};

// One sequence: its query rows [start, start + len), the keys its tokens can see [lo, hi), n in all.
struct PgSeq {
  int start, span, len, n, lo, hi;
};

// b = B is the padding behind the last packed sequence: no keys.  span: tokens whose rows are written (a padded
// batch's sequences hold S rows, of which len are real).  Lengths and prefix sums are clamped before any use.
__device__ __forceinline__ PgSeq pg_seq(const PgArgs& a, int b) {
  PgSeq s;
  if (a.cu_q) {
    const int from = b > 0 ? min(max(a.cu_q[b - 1], 0), a.T) : 0;
    const int to = b < a.B ? min(max(a.cu_q[b], from), a.T) : a.T;
    s.start = from;
    s.span = s.len = to - from;
  } else {
    s.start = b < a.B ? b * a.S : a.T;
    s.span = b < a.B ? a.S : 0;
    s.len = b < a.B && a.q_len ? min(max(a.q_len[b], 0), a.S) : s.span;
  }
  s.n = b < a.B ? min(max(a.kv_len[b], 0), a.max_blocks * a.block_size) : 0;
  s.hi = s.len > 0 ? s.n : 0;
  const int first = s.n - s.len;  // position of the first token
  s.lo = a.win >= 0 && first > a.win ? (first - a.win) & ~(kPgTile - 1) : 0;
  if (s.lo > s.hi) s.lo = s.hi;
  return s;
}

template <int kD>
__host__ __device__ constexpr int pg_swz(int k) {
  // 256-byte rows: see sparse_gqa.hip's layout.  128-byte rows, four to the 512 bytes of all banks: rows r, r + 4,
  // r + 8, r + 12 of a half wave's K operand read take the chunk pairs 0..1, 2..3, 4..5, 6..7.
  return kD == 128 ? 4 * ((k >> 1) & 3) + 2 * ((k >> 3) & 1) : 2 * ((k >> 2) & 3);
}

// Floats of a part: the rows' sums, then their (maximum, sum).
template <int kR, int kD>
__host__ __device__ constexpr int pg_part_floats() { return kR * (kD + 2); }

// j / block_size for 0 <= j < 2^31.  With l = ceil(log2 d) and M = floor(2^(31 + l) / d) + 1, M d exceeds 2^(31 + l) by
// at most 2^l, so j M / 2^(31 + l) exceeds j / d by less than 1 / d and has its whole part.
__device__ __forceinline__ int pg_block(const PgArgs& a, int j) {
  return a.div_mul ? (int)(__umulhi((uint32_t)j, a.div_mul) >> a.div_shift) : j;
}

// Values that a row does not see must not reach it, whatever they hold, but 0 times an infinity or a NaN is a NaN in
// the product of probabilities and V.  So tiles that some row sees in part are searched for such values (unseen
// ones of other tiles do not exist); where there are any, the product takes zeros in their place, and rows that do
// see them get them added by hand.  In tiles that all rows see whole the product takes them as they are: an infinity
// whose weight rounds to 0 gives NaN there and an infinity here, neither of them finite.
// Of a pair of 16-bit values: bit 15 (and 31) set where the value is infinite or NaN: the exponent's ones plus one.
template <bool kF16>
__device__ __forceinline__ uint32_t pg_not_finite(uint32_t w) {
  constexpr uint32_t kOnes = kF16 ? 0x7c007c00u : 0x7f807f80u, kOne = kF16 ? 0x04000400u : 0x00800080u;
  return ((w & kOnes) + kOne) & 0x80008000u;
}
template <bool kF16>
__device__ __forceinline__ void pg_clean(u32x2& v) {
#pragma unroll
  for (int i = 0; i < 2; ++i) v[i] &= ~((pg_not_finite<kF16>(v[i]) >> 15) * 0xffffu);
}
// x where it is not finite, else 0.
template <bool kF16>
__device__ __forceinline__ float pg_only_bad(uint32_t w, int hi) {
  const uint16_t u = (uint16_t)(hi ? w >> 16 : w);
  if (!(pg_not_finite<kF16>(u) & 0x8000u)) return 0.f;
  if constexpr (kF16) return (float)__builtin_bit_cast(_Float16, u);
  else return __uint_as_float((uint32_t)u << 16);
}

// Keys behind a sequence's last one, and of pages outside the pool, load this row: 0 times what lies there need
// not be 0.
static __device__ __align__(128) uint8_t kPgZeroRow[256];

// What becomes of a row's sums o, taken beside the maximum m (base 2), whose weights add up to l: out = o * scale.
// `sink` is -infinity where there is none.  A row that saw nothing (l = 0) has its sink for lse as it is, whatever its
// exponential is.  So has a row whose sink is infinite in base 2: all the weight is the sink's.
struct PgEnd {
  float scale, lse;
};
__device__ __forceinline__ float pg_sink(const PgArgs& a, int head) { return a.sinks ? a.sinks[head] : -kPgInf; }
__device__ __forceinline__ PgEnd pg_end(float m, float l, float sink) {
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
  const float sk = sink * kLog2e, top = fmaxf(m, sk), beside = top == -kPgInf ? 0.f : top;
  const float f = fast_exp2(m - beside), sum = l * f + (sk == kPgInf ? 1.f : fast_exp2(sk - beside));
  const bool only = l == 0.f || (sk == kPgInf && sum == 1.f);
  return {only ? 0.f : f / sum, only ? sink : (beside + fast_log2(sum)) * kLn2};
}

// The keys [k0, k1) of tile `tile` of sequence s, group kvg; `whole`: these are all its keys (the result goes to
// out and lse, otherwise to the part).  Two stages of K and V of 32 keys a wave; the merge reuses a wave's ring, its
// (maximum, sum) lie behind.  Bound by the caches' bytes: 64 tokens over 8192 keys each, 64 heads over 4 of 128: 200 us,
// 5.4 TB/s; one token over 4097: 9 us and the join's 6, latencies.
template <bool kF16, int kD, int kHB>
__device__ __forceinline__ void pg_keys(const PgArgs& a, const PgSeq& s, int b, int tile, int kvg, int k0, int k1,
                                        bool whole, float* part, uint8_t* lds) {
  constexpr int kRow = kD * 2;
  constexpr int kTileBytes = kPgTile * kRow;
  constexpr int kChunks = kD / 8;            // 16-byte chunks of a row
  constexpr int kRpi = kWave / kChunks;      // rows a DMA instruction moves
  constexpr int kInstr = kPgTile / kRpi;     // DMA instructions of a tile
  constexpr int kSt = kD / 32;
  constexpr int kNb = kD / 16;
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane & 15, g = lane >> 4;

  const int rows = s.span * a.Hg;  // of the sequence in this group (T * H < 2^31)
  const int rho0 = tile * 16 * kHB;
  u32x4 qb[kHB][kSt];
  int lim[kHB], low[kHB];  // the row sees keys low .. lim
#pragma unroll
  for (int hb = 0; hb < kHB; ++hb) {
    const int rho = min(rho0 + 16 * hb + r, rows - 1);
    const int i = rho / a.Hg, h = rho - i * a.Hg;
    const uint16_t* qp = a.q + ((int64_t)(s.start + i) * a.H + kvg * a.Hg + h) * kD + 8 * g;
#pragma unroll
    for (int st = 0; st < kSt; ++st) qb[hb][st] = *reinterpret_cast<const u32x4*>(qp + 32 * st);
    const int p = s.n - s.len + i;
    lim[hb] = i < s.len ? (a.causal ? min(p, s.n - 1) : s.n - 1) : -1;
    low[hb] = a.win >= 0 ? max(p, 0) - a.win : 0;
  }
  // Tiles in which every row sees every key skip the comparisons.
  int all_lim = lim[0], all_low = low[0];
#pragma unroll
  for (int hb = 1; hb < kHB; ++hb) {
    all_lim = min(all_lim, lim[hb]);
    all_low = max(all_low, low[hb]);
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    all_lim = min(all_lim, __shfl_xor(all_lim, o, kWave));
    all_low = max(all_low, __shfl_xor(all_low, o, kWave));
  }
  all_lim = __builtin_amdgcn_readfirstlane(all_lim);
  all_low = __builtin_amdgcn_readfirstlane(all_low);

  uint8_t* ring = lds + wave * 4 * kTileBytes;
  const int32_t* bt = a.table + (int64_t)b * a.max_blocks;
  const uint8_t *kb = reinterpret_cast<const uint8_t*>(a.kc), *vb = reinterpret_cast<const uint8_t*>(a.vc);
  // Row of key j in the pools, -1 where there is none.
  auto phys = [&](int j) {
    int row = -1;
    if (j < k1) {
      const int blk = pg_block(a, j), page = bt[blk];
      if (page >= 0 && page < a.num_blocks) row = page * a.block_size + (j - blk * a.block_size);
    }
    return row;
  };
  // DMA of the 32 keys whose rows lie in the lanes' prow (lane l: key l & 31) into stage st.
  const int cpos = lane % kChunks, crow = lane / kChunks;
  auto dma = [&](int prow, int st) {
    uint8_t* dst = ring + st * 2 * kTileBytes;
#pragma unroll
    for (int n = 0; n < kInstr; ++n) {
      const int key = n * kRpi + crow;
      const int rw = __shfl(prow, key, kWave);
      const int64_t at = ((int64_t)rw * a.G + kvg) * kRow + 16 * (cpos ^ pg_swz<kD>(key));
      const uint8_t* zero = kPgZeroRow + 16 * (cpos & 15);
      __builtin_amdgcn_global_load_lds((gqa_gbl_void*)(rw >= 0 ? kb + at : zero), (gqa_lds_void*)(dst + n * 1024), 16,
                                       0, 0);
      __builtin_amdgcn_global_load_lds((gqa_gbl_void*)(rw >= 0 ? vb + at : zero),
                                       (gqa_lds_void*)(dst + kTileBytes + n * 1024), 16, 0, 0);
    }
  };

  uint32_t k_off[kSt], v_off[kSt];
#pragma unroll
  for (int st = 0; st < kSt; ++st) k_off[st] = r * kRow + 16 * ((4 * st + g) ^ pg_swz<kD>(r));
  {
    const int kk = 4 * g + (r >> 2);
#pragma unroll
    for (int p = 0; p < kSt; ++p) v_off[p] = kk * kRow + 16 * ((4 * p + (r & 3)) ^ pg_swz<kD>(kk));
  }
  f32x4 o[kHB][kNb];
  float m_run[kHB], l_run[kHB];
#pragma unroll
  for (int hb = 0; hb < kHB; ++hb) {
#pragma unroll
    for (int i = 0; i < kNb; ++i) o[hb][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m_run[hb] = -kPgInf;
    l_run[hb] = 0.f;
  }

  const int kw = k0 + wave * kPgTile;  // this wave's first key
  const int steps = kw < k1 ? (k1 - kw + kPgUnit - 1) / kPgUnit : 0;
  const int row0 = phys(kw + (lane & 31));
  int next_row = phys(kw + kPgUnit + (lane & 31));
  uint32_t ok_cur = (uint32_t)__ballot(row0 >= 0);
  if (steps > 0) dma(row0, 0);
  for (int e = 0; e < steps; ++e) {
    const int j0 = kw + e * kPgUnit;
    // The rows of the tile after next are looked up ahead of the next tile's DMA, so that waiting for them leaves
    // the DMA in flight.
    const int after = phys(j0 + 2 * kPgUnit + (lane & 31));
    const uint32_t ok_next = (uint32_t)__ballot(next_row >= 0);
    if (e + 1 < steps) dma(next_row, (e + 1) & 1);
    next_row = after;
    if (e + 1 < steps) gqa_wait_vmcnt<2 * kInstr>();
    else gqa_wait_vmcnt<0>();
    const uint32_t base = gqa_lds_u32(ring + (e & 1) * 2 * kTileBytes);
    u32x4 kop[2 * kSt];
    u32x2 vop[kNb][2];
#pragma unroll
    for (int st = 0; st < kSt; ++st) {
      gqa_b128<0>(kop[st], base + k_off[st]);
      gqa_b128<16 * kRow>(kop[kSt + st], base + k_off[st]);
    }
#pragma unroll
    for (int p = 0; p < kSt; ++p) {
      gqa_tr<kTileBytes>(vop[2 * p][0], base + v_off[p]);
      gqa_tr<kTileBytes + 16 * kRow>(vop[2 * p][1], base + v_off[p]);
      gqa_tr<kTileBytes + 8>(vop[2 * p + 1][0], base + v_off[p]);
      gqa_tr<kTileBytes + 16 * kRow + 8>(vop[2 * p + 1][1], base + v_off[p]);
    }
    gqa_lgkm_wait(kop);
#pragma unroll
    for (int i = 0; i < kNb; ++i) __asm__ __volatile__("" : "+v"(vop[i][0]), "+v"(vop[i][1]));

    // S^T: lane (g, r) holds keys j0 + 4 g + i (c[.][0]) and j0 + 16 + 4 g + i (c[.][1]) of row r.
    f32x4 c[kHB][2];
#pragma unroll
    for (int hb = 0; hb < kHB; ++hb)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < kSt; ++st) acc = gqa_mfma<kF16>(kop[k * kSt + st], qb[hb][st], acc);
        c[hb][k] = acc;
      }
    const bool partly = ok_cur != 0xffffffffu || j0 + kPgTile - 1 > all_lim || j0 < all_low;
    if (partly) {
#pragma unroll
      for (int hb = 0; hb < kHB; ++hb)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int kk = 16 * k + 4 * g + i;
            const bool see = ((ok_cur >> kk) & 1u) && j0 + kk <= lim[hb] && j0 + kk >= low[hb];
            c[hb][k][i] = see ? c[hb][k][i] : -kPgInf;
          }
    }
    u32x4 pb[kHB];
#pragma unroll
    for (int hb = 0; hb < kHB; ++hb) {
      float mx = -kPgInf;
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fmaxf(c[hb][0][i], c[hb][1][i]));
      mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
      mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
      const float m_new = fmaxf(m_run[hb], mx * a.scale_log2);  // sm_scale > 0
      const float m_use = m_new == -kPgInf ? 0.f : m_new;
      const float alpha = fast_exp2(m_run[hb] - m_use);
      m_run[hb] = m_new;
      float pv[8], psum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pv[i] = fast_exp2(c[hb][0][i] * a.scale_log2 - m_use);
        pv[4 + i] = fast_exp2(c[hb][1][i] * a.scale_log2 - m_use);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) psum += pv[i];
      l_run[hb] = l_run[hb] * alpha + psum;
#pragma unroll
      for (int i = 0; i < kNb; ++i) o[hb][i] *= alpha;
      pb[hb] = u32x4{gqa_pack<kF16>(pv[0], pv[1]), gqa_pack<kF16>(pv[2], pv[3]), gqa_pack<kF16>(pv[4], pv[5]),
                     gqa_pack<kF16>(pv[6], pv[7])};
    }
    if (partly) {
      uint32_t bad = 0;
#pragma unroll
      for (int i = 0; i < kNb; ++i)
        bad |= pg_not_finite<kF16>(vop[i][0].x) | pg_not_finite<kF16>(vop[i][0].y) | pg_not_finite<kF16>(vop[i][1].x) |
               pg_not_finite<kF16>(vop[i][1].y);
      if (__any(bad != 0)) {
#pragma unroll
        for (int i = 0; i < kNb; ++i) {
          pg_clean<kF16>(vop[i][0]);
          pg_clean<kF16>(vop[i][1]);
        }
        const uint8_t* vt = ring + (e & 1) * 2 * kTileBytes + kTileBytes;
        for (int j = 0; j < kPgTile; ++j) {
          if (!((ok_cur >> j) & 1u)) continue;
#pragma unroll
          for (int p = 0; p < kSt; ++p) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(vt + j * kRow + 16 * ((4 * p + g) ^ pg_swz<kD>(j)));
#pragma unroll
            for (int hb = 0; hb < kHB; ++hb) {
              const bool see = j0 + j <= lim[hb] && j0 + j >= low[hb];
#pragma unroll
              for (int i = 0; i < 8; ++i) o[hb][2 * p + (i >> 2)][i & 3] += see ? pg_only_bad<kF16>(w[i / 2], i & 1) : 0.f;
            }
          }
        }
      }
    }
    // O^T += V^T P^T: lane (g, r) of block 2p + h accumulates row r, columns 32 p + 8 g + 4 h .. + 3.
#pragma unroll
    for (int i = 0; i < kNb; ++i) {
      const u32x4 va = {vop[i][0].x, vop[i][0].y, vop[i][1].x, vop[i][1].y};
#pragma unroll
      for (int hb = 0; hb < kHB; ++hb) o[hb][i] = gqa_mfma<kF16>(va, pb[hb], o[hb][i]);
    }
    ok_cur = ok_next;
  }

  // Merge of the waves.
  __builtin_amdgcn_s_waitcnt(0);
  float* ow = reinterpret_cast<float*>(ring);  // [16 kHB][kD]
  float* ml = reinterpret_cast<float*>(lds + kPgWaves * 4 * kTileBytes);
#pragma unroll
  for (int hb = 0; hb < kHB; ++hb) {
    float l = l_run[hb];
    l += __shfl_xor(l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);
#pragma unroll
    for (int i = 0; i < kNb; ++i)
      *reinterpret_cast<f32x4*>(ow + (16 * hb + r) * kD + 32 * (i / 2) + 8 * g + 4 * (i % 2)) = o[hb][i];
    if (g == 0) {
      ml[(wave * 16 * kHB + 16 * hb + r) * 2] = m_run[hb];
      ml[(wave * 16 * kHB + 16 * hb + r) * 2 + 1] = l;
    }
  }
  __syncthreads();
  constexpr int kPerRow = kD / 8;                  // threads of a row
  constexpr int kRowsPass = kPgThreads / kPerRow;  // 16 or 32
#pragma unroll
  for (int r0 = 0; r0 < 16 * kHB; r0 += kRowsPass) {
    const int hh = r0 + tid / kPerRow, c0 = 8 * (tid % kPerRow);
    if (hh >= 16 * kHB) break;
    float mw[kPgWaves], M = -kPgInf;
#pragma unroll
    for (int w = 0; w < kPgWaves; ++w) {
      mw[w] = ml[(w * 16 * kHB + hh) * 2];
      M = fmaxf(M, mw[w]);
    }
    const float M_use = M == -kPgInf ? 0.f : M;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kPgWaves; ++w) {
      const float f = fast_exp2(mw[w] - M_use);
      sum += f * ml[(w * 16 * kHB + hh) * 2 + 1];
      const float* src = reinterpret_cast<const float*>(lds + w * 4 * kTileBytes) + hh * kD + c0;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += f * src[i];
    }
    const int rho = rho0 + hh;
    if (!whole) {
      float* p = part + hh * kD + c0;
      *reinterpret_cast<f32x4*>(p) = f32x4{acc[0], acc[1], acc[2], acc[3]};
      *reinterpret_cast<f32x4*>(p + 4) = f32x4{acc[4], acc[5], acc[6], acc[7]};
      if (c0 == 0) {
        part[16 * kHB * kD + 2 * hh] = M;
        part[16 * kHB * kD + 2 * hh + 1] = sum;
      }
    } else if (rho < rows) {
      const int i = rho / a.Hg, h = kvg * a.Hg + rho - i * a.Hg;
      const int64_t orow = (int64_t)(s.start + i) * a.H + h;
      const PgEnd e = pg_end(M, sum, pg_sink(a, h));
      const float inv = e.scale;
      *reinterpret_cast<u32x4*>(a.out + orow * kD + c0) =
          u32x4{gqa_pack<kF16>(acc[0] * inv, acc[1] * inv), gqa_pack<kF16>(acc[2] * inv, acc[3] * inv),
                gqa_pack<kF16>(acc[4] * inv, acc[5] * inv), gqa_pack<kF16>(acc[6] * inv, acc[7] * inv)};
      if (c0 == 0) a.lse[orow] = e.lse;
    }
  }
  __syncthreads();  // the rings are free for the next item
}

// LDS position of 16-byte chunk c of key k of pg_rows' tiles is c ^ pr_swz(k).  K operand reads (a half wave: 32 keys,
// one chunk) meet each position of the 512 bytes of all banks once: bits 1 to 4 of the key (256-byte rows) or 2 to 4
// (128-byte rows) go to different chunks.  Transposed V reads (8 keys, 64 bytes of each) do too: the upper chunk bits
// come from the keys' low bits.
template <int kD>
__host__ __device__ constexpr int pr_swz(int k) {
  return (kD == 128 ? 4 * ((k >> 1) & 3) : 4 * ((k >> 2) & 1)) + ((k >> 3) & 3);
}

template <bool kF16>
__device__ __forceinline__ f32x16 pr_mfma(const u32x4& a, const u32x4& b, const f32x16& c) {
  if constexpr (kF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}

// All but the kLeft youngest LDS reads have returned; v passes through so that no use moves above the wait.
template <int kLeft, int N, typename V>
__device__ __forceinline__ void pr_lds_wait(V (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) __asm__ __volatile__("" : "+v"(v[i]));
  __asm__ __volatile__("s_waitcnt lgkmcnt(%0)" ::"i"(kLeft) : "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) __asm__ __volatile__("" : "+v"(v[i]));
}

// The larger of x here and in the lane 32 away.
__device__ __forceinline__ float pr_max32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pr_sum32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// f(integral_constant) for kFrom .. kTo - 1.
template <int kFrom, int kTo, class F>
__device__ __forceinline__ void pr_each(F&& f) {
  if constexpr (kFrom < kTo) {
    f(std::integral_constant<int, kFrom>{});
    pr_each<kFrom + 1, kTo>(f);
  }
}

constexpr int kPrWaves = 8;
constexpr int kPrThreads = kPrWaves * kWave;
constexpr int kPrRows = 32 * kPrWaves;  // 256
constexpr int kPrTile = 64;             // keys

// As pg_keys, for 256 rows.  Body t of a wave is C(t): scores of tile t and the products of tile t - 1 with V, a
// barrier, X(t): exponentials of tile t, a barrier; waves 4 to 7 run one barrier behind, so that on each SIMD one
// wave is in C while the other is in X.  Rings of four stages: C(t) starts the DMA of K of tile t + 3 and V of tile
// t + 2, into the stages of K(t - 1) and V(t - 2), whose last reads (in C(t - 1) of the later waves) lie before the
// barrier ahead of C(t) of the earlier ones.  The wait at the end of C(t) leaves only what C(t) started in flight:
// behind two barriers more K(t + 2) and V(t + 1) are whole, so that X(t) may begin with the first reads of C(t + 1).
// 64-wide heads have one barrier a body instead of two, the halves still apart: between two barriers waves 0 to 3 have
// C(t) and X(t), waves 4 to 7 X(t - 1) and C(t).  Those read K(t), K(t + 1), V(t - 1) and V(t), whole by the wait at
// the end of C(t - 1) and the barrier behind it, and the DMA of C(t) goes to K(t - 1) and V(t - 2), last read before
// that barrier.  16K prompts, 64 heads over 4: 2697 -> 2593 us; 128-wide heads 3970 -> 4152; both halves in phase: 4409.
// 128-wide heads reach 1123 TFLOP/s there (3915 us, 3875 to 4010 by card); 512 tokens over 65536 keys 1038 us, 1055;
// 64-wide heads 878 at the prompt (2504 us).  A tile's LDS reads (64 +
// 64 KB by eight waves) take about 70% of a body's time.
template <bool kF16, int kD, bool kEven>
__device__ __forceinline__ void pg_rows(const PgArgs& a, const PgSeq& s, int b, int tile, int kvg, int k0, int k1,
                                        bool whole, float* part, uint8_t* lds) {
  constexpr int kRow = kD * 2;
  constexpr int kTileBytes = kPrTile * kRow;
  constexpr int kChunks = kD / 8;
  constexpr int kRpi = kWave / kChunks;               // rows a DMA instruction moves
  constexpr int kI = kPrTile / kRpi / kPrWaves;       // DMA instructions of a wave and tile
  constexpr int kSt = kD / 16;                        // steps of the score product
  constexpr int kNb = kD / 32;                        // 32-column blocks of the output
  constexpr bool kOne = kD == 64;                     // one barrier a body (64 KB of LDS reads a tile, not 128)
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane & 31, hi = lane >> 5;

  const int rows = s.span * a.Hg;
  const int first = tile * kPrRows + 32 * wave;
  const int rho = min(first + r, rows - 1);
  const int tok = rho / a.Hg, head = kvg * a.Hg + rho - tok * a.Hg;
  const int64_t qrow = (int64_t)(s.start + tok) * a.H + head;
  // Q operand (B): row r, dims 16 st + 8 hi .. + 7.
  u32x4 qb[kSt];
#pragma unroll
  for (int st = 0; st < kSt; ++st) qb[st] = *reinterpret_cast<const u32x4*>(a.q + qrow * kD + 16 * st + 8 * hi);
  const int pos = s.n - s.len + tok;
  const int lim = tok < s.len ? (a.causal ? min(pos, s.n - 1) : s.n - 1) : -1;  // the row sees keys low .. lim
  const int low = a.win >= 0 ? max(pos, 0) - a.win : 0;
  int lim_min = lim, low_max = low;  // tiles in which every row sees every key skip the comparisons
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    lim_min = min(lim_min, __shfl_xor(lim_min, o, kWave));
    low_max = max(low_max, __shfl_xor(low_max, o, kWave));
  }
  lim_min = __builtin_amdgcn_readfirstlane(lim_min);
  low_max = __builtin_amdgcn_readfirstlane(low_max);
  // Tiles of keys in [part_lo, part_hi] are seen whole by every token of the workgroup's rows.
  const int tok0 = tile * kPrRows / a.Hg, tok1 = min(((tile + 1) * kPrRows - 1) / a.Hg, s.len - 1);
  const int part_hi = a.causal ? min(s.n - s.len + tok0, s.n - 1) : s.n - 1;
  const int part_lo = a.win >= 0 ? max(s.n - s.len + tok1, 0) - a.win : 0;

  f32x16 o[kNb];
#pragma unroll
  for (int p = 0; p < kNb; ++p)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[p][i] = 0.f;
  float m_run = -kPgInf, l_run = 0.f;

  const int32_t* bt = a.table + (int64_t)b * a.max_blocks;
  const int nt = k1 > k0 ? (k1 - k0 + kPrTile - 1) / kPrTile : 0;
  if (nt > 0) {
    // Pages outside the pool hide their keys: looked for once, the comparisons look again where there are any.  The
    // first load of a thread is judged behind the first DMA.
    const int last_blk = pg_block(a, k1 - 1), my_blk = pg_block(a, k0) + tid;
    const int my_page = bt[min(my_blk, last_blk)];
    int outside = 0;
    for (int blk = my_blk + kPrThreads; blk <= last_blk; blk += kPrThreads)
      outside |= (uint32_t)bt[blk] >= (uint32_t)a.num_blocks;

    const uint8_t *kb = reinterpret_cast<const uint8_t*>(a.kc), *vb = reinterpret_cast<const uint8_t*>(a.vc);
    const int crow = lane / kChunks, cpos = lane % kChunks;
    const uint8_t* zero = kPgZeroRow + 16 * (cpos & 15);
    // DMA instruction i of a wave moves kRpi keys from key first_key(t, i) on; chunk positions repeat every 32 keys.
    const int swz = 16 * (cpos ^ pr_swz<kD>(wave * kRpi + crow));
    auto first_key = [&](int t, int i) { return k0 + t * kPrTile + (wave + kPrWaves * i) * kRpi; };
    auto to_lds = [&](const uint8_t* src, int ring, int t, int i) {
      __builtin_amdgcn_global_load_lds((gqa_gbl_void*)src,
                                       (gqa_lds_void*)(lds + (4 * ring + (t & 3)) * kTileBytes + (wave + kPrWaves * i) * 1024),
                                       16, 0, 0);
    };
    // Where the keys of an instruction lie.  kEven: in one page (block_size is a multiple of 8, k0 of 32), whose number
    // is a scalar load; the row is that of the first key, -1 without a page, `left` the keys before k1.
    // Otherwise each lane looks up its own key (a load without a condition), and the row is the lane's, -1 without a key.
    struct Look {
      int page, rem, left;
    };
    struct Place {
      int row, left;
    };
    auto look = [&](int t, int i) {
      const int j = first_key(t, i) + (kEven ? 0 : crow), jc = min(j, k1 - 1), blk = pg_block(a, jc);
      typedef const __attribute__((address_space(4))) int32_t const_i32;
      const int page = kEven ? *(const_i32*)(bt + __builtin_amdgcn_readfirstlane(blk)) : bt[blk];
      return Look{page, jc - blk * a.block_size, k1 - j};
    };
    auto place = [&](const Look& l) {
      const bool ok = l.left > 0 && (uint32_t)l.page < (uint32_t)a.num_blocks;
      return Place{ok ? l.page * a.block_size + l.rem : -1, l.left};
    };
    const int64_t row_bytes = (int64_t)a.G * kRow;
    const int lane_off = crow * a.G * kRow + swz;
    auto dma = [&](const uint8_t* cache, const Place& p, int ring, int t, int i) {
      const uint8_t* base = cache + p.row * row_bytes + kvg * kRow;
      if constexpr (kEven) to_lds(p.row >= 0 && crow < p.left ? base + lane_off : zero, ring, t, i);
      else to_lds(p.row >= 0 ? base + swz : zero, ring, t, i);
    };
    Place knext[kI], vnext[kI];  // of tiles t + 3 and t + 2
    {
      Place at0[kI], at1[kI];
#pragma unroll
      for (int i = 0; i < kI; ++i) {
        at0[i] = place(look(0, i));
        at1[i] = place(look(1, i));
        vnext[i] = place(look(2, i));
        knext[i] = place(look(3, i));
      }
#pragma unroll
      for (int i = 0; i < kI; ++i) dma(kb, at0[i], 0, 0, i);
#pragma unroll
      for (int i = 0; i < kI; ++i) dma(vb, at0[i], 1, 0, i);
#pragma unroll
      for (int i = 0; i < kI; ++i) dma(kb, at1[i], 0, 1, i);
#pragma unroll
      for (int i = 0; i < kI; ++i) dma(vb, at1[i], 1, 1, i);
#pragma unroll
      for (int i = 0; i < kI; ++i) dma(kb, vnext[i], 0, 2, i);
    }
    auto dma_k = [&](int t) {
#pragma unroll
      for (int i = 0; i < kI; ++i) dma(kb, knext[i], 0, t + 3, i);
    };
    auto dma_v = [&](int t) {
#pragma unroll
      for (int i = 0; i < kI; ++i) {
        dma(vb, vnext[i], 1, t + 2, i);
        vnext[i] = knext[i];
      }
    };

    // Where K of tile t + 4 lies: asked at the start of C(t), taken at its end.
    Look asked[kI];
    auto ask = [&](int t) {
#pragma unroll
      for (int i = 0; i < kI; ++i) asked[i] = look(t + 4, i);
    };
    auto take = [&] {
#pragma unroll
      for (int i = 0; i < kI; ++i) knext[i] = place(asked[i]);
    };

    const uint32_t lds0 = gqa_lds_u32(lds);
    // K operand (A), step st, key block kb: key 32 kb + r, dims 16 st + 8 hi .. + 7.
    const uint32_t k_at = lds0 + r * kRow + 16 * (hi ^ pr_swz<kD>(r));
    // V^T operand (A), 16 keys from 16 u, columns 32 p ..: lane group (hi, h) of 16 lanes (q = lane & 15) addresses
    // keys 4 hi + (q >> 2) (+ 8 for the second read), columns 16 h + 8 (q & 1) + 4 ((q >> 1) & 1) .. + 3, and receives
    // those keys of one column each: operand row 16 h + 4 c + e is column 16 h + 8 (c & 1) + 4 (c >> 1) + e, so that
    // a lane's results 8 x .. 8 x + 7 are columns 16 x + 8 hi .. + 7.
    const int q = lane & 15, h = (lane >> 4) & 1, vk = 4 * hi + (q >> 2);
    const uint32_t v_at =
        lds0 + 4 * kTileBytes + vk * kRow + 16 * ((2 * h + (q & 1)) ^ pr_swz<kD>(vk)) + 8 * ((q >> 1) & 1);

    // A body's LDS reads, in batches of four: batches 0 .. kNk - 1 the K operands of two steps of both key blocks, then
    // the V operands of two column blocks and 16 keys.  Three batches are in flight ahead of the one multiplied.
    constexpr int kNk = kSt / 2, kNv = 2 * kNb;
    u32x4 kop[kNk][4];
    u32x2 vop[kNv][4];
    u32x4 pb[4];
    f32x16 c[2];
    auto read = [&](int t, auto batch) {
      constexpr int i = decltype(batch)::value;
      if constexpr (i < kNk) {
        const uint32_t at = k_at + (t & 3) * kTileBytes;
        gqa_b128<0>(kop[i][0], at ^ (64 * i));
        gqa_b128<32 * kRow>(kop[i][1], at ^ (64 * i));
        gqa_b128<0>(kop[i][2], at ^ (64 * i + 32));
        gqa_b128<32 * kRow>(kop[i][3], at ^ (64 * i + 32));
      } else {
        constexpr int u = (i - kNk) / (kNb / 2), p = 2 * ((i - kNk) % (kNb / 2));
        const uint32_t at = v_at + ((t - 1) & 3) * kTileBytes;
        gqa_tr<16 * u * kRow>(vop[i - kNk][0], at ^ (64 * p + 16 * ((2 * u) & 3)));
        gqa_tr<(16 * u + 8) * kRow>(vop[i - kNk][1], at ^ (64 * p + 16 * ((2 * u + 1) & 3)));
        gqa_tr<16 * u * kRow>(vop[i - kNk][2], at ^ (64 * p + 64 + 16 * ((2 * u) & 3)));
        gqa_tr<(16 * u + 8) * kRow>(vop[i - kNk][3], at ^ (64 * p + 64 + 16 * ((2 * u + 1) & 3)));
      }
    };
    auto mul = [&](auto batch) {
      constexpr int i = decltype(batch)::value;
      if constexpr (i < kNk) {
        if constexpr (i == 0) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) c[k][e] = 0.f;
        }
        c[0] = pr_mfma<kF16>(kop[i][0], qb[2 * i], c[0]);
        c[1] = pr_mfma<kF16>(kop[i][1], qb[2 * i], c[1]);
        c[0] = pr_mfma<kF16>(kop[i][2], qb[2 * i + 1], c[0]);
        c[1] = pr_mfma<kF16>(kop[i][3], qb[2 * i + 1], c[1]);
      } else {
        constexpr int u = (i - kNk) / (kNb / 2), p = 2 * ((i - kNk) % (kNb / 2));
        const u32x2(&v)[4] = vop[i - kNk];
        o[p] = pr_mfma<kF16>(u32x4{v[0].x, v[0].y, v[1].x, v[1].y}, pb[u], o[p]);
        o[p + 1] = pr_mfma<kF16>(u32x4{v[2].x, v[2].y, v[3].x, v[3].y}, pb[u], o[p + 1]);
      }
    };
    // C(t) takes a batch of scores and two of products in turn, so that the transposing reads, the slowest, are spread
    // over all its products: n-th batch.
    const auto nth = [](int n) constexpr { return n % 3 == 0 ? n / 3 : kNk + n - n / 3 - 1; };
    static_assert(kNv == 2 * kNk, "a batch of scores and two of products in turn");
    auto wait_for = [&](auto left, auto batch) {
      constexpr int i = decltype(batch)::value;
      if constexpr (i < kNk) pr_lds_wait<decltype(left)::value>(kop[i]);
      else pr_lds_wait<decltype(left)::value>(vop[i - kNk]);
    };
    auto start = [&](int t) {  // the first three batches of C(t)
      read(t, std::integral_constant<int, nth(0)>{});
      read(t, std::integral_constant<int, nth(1)>{});
      read(t, std::integral_constant<int, nth(2)>{});
    };
    auto body = [&](int t) {
      ask(t);
      constexpr int kAll = kNk + kNv;
      pr_each<0, kAll>([&](auto i) {
        // Twelve reads are out: the counter of them holds fifteen.
        constexpr int n = decltype(i)::value, left = kAll - 1 - n < 2 ? kAll - 1 - n : 2;
        wait_for(std::integral_constant<int, 4 * left>{}, std::integral_constant<int, nth(n)>{});
        if constexpr (n + 3 < kAll) read(t, std::integral_constant<int, nth(n + 3)>{});
        mul(std::integral_constant<int, nth(n)>{});
        if constexpr (n == 0) dma_k(t);
        if constexpr (n == 1) dma_v(t);
      });
      take();
    };
    auto products_only = [&](int t) {  // of tile t - 1
      pr_each<kNk, kNk + 3>([&](auto i) { read(t, i); });
      pr_each<kNk, kNk + kNv>([&](auto i) {
        constexpr int n = decltype(i)::value, left = kNk + kNv - 1 - n < 2 ? kNk + kNv - 1 - n : 2;
        wait_for(std::integral_constant<int, 4 * left>{}, i);
        if constexpr (n + 3 < kNk + kNv) read(t, std::integral_constant<int, n + 3>{});
        mul(i);
      });
    };
    auto scores_only = [&](int t) {
      read(t, std::integral_constant<int, 0>{});
      read(t, std::integral_constant<int, 1>{});
      ask(t);
      pr_each<0, kNk>([&](auto i) {
        constexpr int n = decltype(i)::value;
        pr_lds_wait<n + 1 < kNk ? 4 : 0>(kop[n]);
        if constexpr (n + 2 < kNk) read(t, std::integral_constant<int, n + 2>{});
        mul(i);
      });
      dma_k(t);
      dma_v(t);
      take();
    };
    const auto turn = [] { __builtin_amdgcn_s_barrier(); };
    gqa_wait_vmcnt<(kOne ? 2 : 3) * kI>();
    // The waves' findings pass through LDS by hand: a fence or a plain access would wait for the DMA.
    const uint32_t flags = gqa_lds_u32(lds + 8 * kTileBytes);
    const bool found = __any(outside | ((uint32_t)my_page >= (uint32_t)a.num_blocks));
    __asm__ __volatile__("ds_write_b8 %0, %1\n\ts_waitcnt lgkmcnt(0)" ::"v"(flags + 16 + wave), "v"((int)found)
                         : "memory");
    turn();
    u32x2 seen;
    __asm__ __volatile__("ds_read_b64 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(seen) : "v"(flags + 16) : "memory");
    const bool holes = __builtin_amdgcn_readfirstlane((int)(seen.x | seen.y)) != 0;
    auto softmax = [&](int t) {
      const int j0 = k0 + t * kPrTile;
      if (holes || j0 + kPrTile - 1 > lim_min || j0 < low_max) {
        uint64_t there = ~(uint64_t)0;  // keys in pages of the pool
        if (holes) there = __ballot((uint32_t)bt[pg_block(a, min(j0 + lane, k1 - 1))] < (uint32_t)a.num_blocks);
        const int up = lim - j0 - 4 * hi, down = low - j0 - 4 * hi;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t bits = (uint32_t)(there >> (32 * k)) >> (4 * hi);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int j = 8 * (i >> 2) + (i & 3);
            const bool see = 32 * k + j <= up && 32 * k + j >= down && ((bits >> j) & 1u);
            c[k][i] = see ? c[k][i] : -kPgInf;
          }
        }
      }
      // `maximum` needs no quieting of its operands beforehand, as fmaxf does: v_maximum3_f32.
      float mx = __builtin_elementwise_maximum(c[0][0], c[1][0]);
#pragma unroll
      for (int i = 1; i < 16; ++i)
        mx = __builtin_elementwise_maximum(__builtin_elementwise_maximum(mx, c[0][i]), c[1][i]);
      mx = pr_max32(mx) * a.scale_log2;  // sm_scale > 0
      // The reference moves only when it falls 2^8 behind: a probability is at most 2^8 then, in the range of every
      // type here, and most tiles leave the sums as they are.
      if (__any(mx > m_run + 8.f)) {
        const float m_new = fmaxf(m_run, mx);
        const float alpha = m_new == -kPgInf ? 1.f : fast_exp2(m_run - m_new);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int p = 0; p < kNb; ++p) o[p] *= alpha;
      }
      const float m_use = m_run == -kPgInf ? 0.f : m_run;
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          c[k][i] = fast_exp2(fmaf(c[k][i], a.scale_log2, -m_use));
          sum += c[k][i];
        }
      l_run += sum;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int x = 8 * (u & 1);
        const f32x16& e = c[u >> 1];
        pb[u] = u32x4{gqa_pack<kF16>(e[x], e[x + 1]), gqa_pack<kF16>(e[x + 2], e[x + 3]),
                      gqa_pack<kF16>(e[x + 4], e[x + 5]), gqa_pack<kF16>(e[x + 6], e[x + 7])};
      }
    };
    const bool late = wave >= 4;
    // V of tile t, searched for values that are not finite where some row sees the tile in part: two barriers ahead of
    // its first use, an eighth by each wave, which notes what it found; one barrier later they are replaced by zeros
    // in LDS, by every wave (one that reads ahead in the same turn reads its own zeros).  What the rows do see of
    // them is added behind the loop.  Tiles [part_end, part_begin) are seen whole by all rows.
    const int part_end = part_lo > k0 ? min((part_lo - k0 + kPrTile - 1) / kPrTile, nt) : 0;
    const int part_begin = part_hi + 1 > k0 ? min((part_hi + 1 - k0) / kPrTile, nt) : 0;
    const auto in_part = [&](int t) { return t < nt && (t < part_end || t >= part_begin); };
    bool any_bad = false;
    auto search = [&](int t) {
      if (!in_part(t)) return;
      const uint32_t at = lds0 + (4 + (t & 3)) * kTileBytes + wave * (kTileBytes / kPrWaves) + 16 * lane;
      u32x4 w[kTileBytes / kPrWaves / 1024];
      __asm__ __volatile__("s_waitcnt lgkmcnt(0)" ::: "memory");
      gqa_b128<0>(w[0], at);
      if constexpr (kTileBytes / kPrWaves == 2048) gqa_b128<1024>(w[1], at);
      gqa_lgkm_wait(w);
      uint32_t bad = 0;
#pragma unroll
      for (int n = 0; n < kTileBytes / kPrWaves / 1024; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= pg_not_finite<kF16>(w[n][i]);
      const int note = __any(bad != 0);
      __asm__ __volatile__("ds_write_b8 %0, %1\n\ts_waitcnt lgkmcnt(0)" ::"v"(flags + 8 * (t & 1) + wave), "v"(note)
                           : "memory");
    };
    auto scrub = [&](int t) {
      if (!in_part(t)) return;
      u32x2 notes;
      __asm__ __volatile__("ds_read_b64 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(notes) : "v"(flags + 8 * (t & 1)) : "memory");
      if (__builtin_amdgcn_readfirstlane((int)(notes.x | notes.y)) == 0) return;
      any_bad = true;
      uint8_t* vt = lds + (4 + (t & 3)) * kTileBytes + 8 * lane;
#pragma unroll 1
      for (int n = 0; n < kTileBytes; n += 512) {
        u32x2 w = *reinterpret_cast<u32x2*>(vt + n);
        pg_clean<kF16>(w);
        *reinterpret_cast<u32x2*>(vt + n) = w;
      }
      __asm__ __volatile__("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    // Bodies t0 .. t1 - 1 behind C(0) and X(0); without `checked` no tile t0 .. t1 is seen in part.
    auto bodies = [&](int t0, int t1, auto checked) {
      constexpr bool kChecked = decltype(checked)::value;
      for (int t = t0; t < t1; ++t) {
        turn();
        if (kChecked && late) scrub(t);
        __builtin_amdgcn_s_setprio(1);
        body(t);
        __builtin_amdgcn_s_setprio(0);
        gqa_wait_vmcnt<2 * kI>();
        if (kChecked && !late) search(t);
        turn();
        if (kChecked && !late) scrub(t);
        // The first reads of C(t + 1) go out ahead of the exponentials, while the SIMD's other wave is in C.
        start(t + 1);
        softmax(t);
        if (kChecked && late) search(t + 1);
      }
    };
    const auto drop = [&] {  // the reads of a tile behind the last
      wait_for(std::integral_constant<int, 0>{}, std::integral_constant<int, nth(0)>{});
      wait_for(std::integral_constant<int, 0>{}, std::integral_constant<int, nth(1)>{});
      wait_for(std::integral_constant<int, 0>{}, std::integral_constant<int, nth(2)>{});
    };
    const int whole0 = max(part_end, 1), whole1 = max(part_begin - 1, whole0);
    if (first < rows) {
      if constexpr (kOne) {
        // A tile seen in part is searched and cleaned behind its turn, with a barrier between.
        const auto check = [&](int t) {
          if (!in_part(t)) return;
          search(t);
          turn();
          scrub(t);
        };
        // Bodies as below, one turn each: before C(t) of waves 0 to 3, between C(t - 1) and X(t - 1) of the others.
        const auto rest = [&](int t, auto checked) {  // of body t, behind C(t)
          gqa_wait_vmcnt<2 * kI>();
          if (late) {
            turn();
            if (decltype(checked)::value) check(t + 1);
          }
          start(t + 1);
          softmax(t);
          if (!late) {
            turn();
            if (decltype(checked)::value) check(t + 1);
          }
        };
        check(0);
        scores_only(0);
        rest(0, std::true_type{});
        const auto run = [&](int t0, int t1, auto checked) {
          for (int t = t0; t < t1; ++t) {
            __builtin_amdgcn_s_setprio(1);
            body(t);
            __builtin_amdgcn_s_setprio(0);
            rest(t, checked);
          }
        };
        run(1, min(whole0, nt), std::true_type{});
        run(whole0, min(whole1, nt), std::false_type{});
        run(max(whole1, 1), nt, std::true_type{});
        drop();
      } else {
        if (late) {
          search(0);
          turn();
          scrub(0);
        }
        scores_only(0);
        gqa_wait_vmcnt<2 * kI>();
        if (!late) search(0);
        turn();
        if (!late) scrub(0);
        start(1);
        softmax(0);
        if (late) search(1);
        bodies(1, min(whole0, nt), std::true_type{});
        bodies(whole0, min(whole1, nt), std::false_type{});
        bodies(max(whole1, 1), nt, std::true_type{});
        drop();
        turn();
      }
      products_only(nt);
      if (any_bad) {
        for (int t = 0; t < nt; ++t) {
          if (!in_part(t)) continue;
          for (int j = k0 + t * kPrTile; j < min(k0 + (t + 1) * kPrTile, k1); ++j) {
            const int blk = pg_block(a, j), page = bt[blk];
            if ((uint32_t)page >= (uint32_t)a.num_blocks) continue;
            const uint8_t* vr = vb + (page * a.block_size + j - blk * a.block_size) * row_bytes + kvg * kRow;
            const bool see = j <= lim && j >= low;
#pragma unroll
            for (int p = 0; p < kNb; ++p)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(vr + 16 * (4 * p + 2 * x + hi));
#pragma unroll
                for (int i = 0; i < 8; ++i) o[p][8 * x + i] += see ? pg_only_bad<kF16>(w[i / 2], i & 1) : 0.f;
              }
          }
        }
      }
    } else {  // no rows: this wave only moves tiles and searches its part of them
      if (!kOne && late) {
        search(0);
        turn();
      }
      for (int t = 0; kOne && t < nt; ++t) {
        if (t > 0) turn();
        if (in_part(t)) {
          search(t);
          turn();
        }
        ask(t);
        dma_k(t);
        dma_v(t);
        take();
        gqa_wait_vmcnt<2 * kI>();
      }
      if (kOne) turn();
      for (int t = 0; !kOne && t < nt; ++t) {
        ask(t);
        dma_k(t);
        dma_v(t);
        take();
        gqa_wait_vmcnt<2 * kI>();
        if (!late) search(t);
        turn();
        if (late) search(t + 1);
        turn();
      }
    }
    if (!kOne && !late) turn();
    __builtin_amdgcn_s_waitcnt(0);  // the DMA of tiles behind the last
  }

  l_run = pr_sum32(l_run);
  const bool none = l_run == 0.f;  // a row that saw nothing: its sums may be 0 times anything
  if (!whole) {
    float* p = part + (32 * wave + r) * kD + 8 * hi;
#pragma unroll
    for (int n = 0; n < kNb; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        *reinterpret_cast<f32x4*>(p + 32 * n + 16 * (x >> 1) + 4 * (x & 1)) =
            none ? f32x4{0.f, 0.f, 0.f, 0.f} : f32x4{o[n][4 * x], o[n][4 * x + 1], o[n][4 * x + 2], o[n][4 * x + 3]};
    if (hi == 0) {
      part[kPrRows * kD + 2 * (32 * wave + r)] = m_run;
      part[kPrRows * kD + 2 * (32 * wave + r) + 1] = l_run;
    }
  } else if (first + r < rows) {
    const PgEnd e = pg_end(m_run, l_run, pg_sink(a, head));
    const float inv = e.scale;
    uint16_t* dst = a.out + qrow * kD + 8 * hi;
#pragma unroll
    for (int n = 0; n < kNb; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = none ? 0.f : o[n][8 * x + i] * inv;
        *reinterpret_cast<u32x4*>(dst + 32 * n + 16 * x) = u32x4{gqa_pack<kF16>(v[0], v[1]), gqa_pack<kF16>(v[2], v[3]),
                                                                gqa_pack<kF16>(v[4], v[5]), gqa_pack<kF16>(v[6], v[7])};
      }
    if (hi == 0) a.lse[qrow] = e.lse;
  }
}

// The two ways with their sizes.
template <bool kF16_, int kD_, int kHB>
struct PgKeys {
  static constexpr bool kF16 = kF16_;
  static constexpr int kD = kD_, kR = 16 * kHB, kUnitKeys = kPgUnit, kThreads = kPgThreads;
  static constexpr int kLds = kPgWaves * 2 * 2 * kPgTile * kD * 2 + kPgWaves * 16 * kHB * 2 * 4;
  static_assert(16 * kHB * kD * 4 <= 4 * kPgTile * kD * 2, "a wave's sums fit its ring");
  static __device__ __forceinline__ void item(const PgArgs& a, const PgSeq& s, int b, int tile, int kvg, int k0, int k1,
                                              bool whole, float* part, uint8_t* lds) {
    pg_keys<kF16, kD, kHB>(a, s, b, tile, kvg, k0, k1, whole, part, lds);
  }
};
template <bool kF16_, int kD_, bool kEven>
struct PgRows {
  static constexpr bool kF16 = kF16_;
  static constexpr int kD = kD_, kR = kPrRows, kUnitKeys = kPrTile, kThreads = kPrThreads;
  static constexpr int kLds = 8 * kPrTile * kD * 2 + 32;  // two rings of four stages, the waves' notes
  static __device__ __forceinline__ void item(const PgArgs& a, const PgSeq& s, int b, int tile, int kvg, int k0, int k1,
                                              bool whole, float* part, uint8_t* lds) {
    pg_rows<kF16, kD, kEven>(a, s, b, tile, kvg, k0, k1, whole, part, lds);
    __syncthreads();  // the rings are free for the next item
  }
};

// First slot of sequence b, whose rows start at `start`: strictly increasing in b.
__device__ __forceinline__ int pg_slot(int start, int Hg, int b, int kR) {
  return (int)((int64_t)start * Hg / kR) + b;
}
// First query row of sequence b; `cu` is a.cu_q or a copy.
__device__ __forceinline__ int pg_start(const PgArgs& a, const int32_t* cu, int b) {
  if (!a.cu_q) return min(b, a.B) * a.S;
  return b > 0 ? min(max(cu[b - 1], 0), a.T) : 0;
}
// The last sequence whose first slot is not past `slot`.
__device__ __forceinline__ int pg_find(const PgArgs& a, const int32_t* cu, int slot, int kR) {
  int b0 = 0, b1 = a.B;
  while (b0 < b1) {
    const int mid = (b0 + b1 + 1) >> 1;
    if (pg_slot(pg_start(a, cu, mid), a.Hg, mid, kR) <= slot) b0 = mid;
    else b1 = mid - 1;
  }
  return b0;
}
// The keys [lo, hi) that rows of the tile see, none for a tile that holds padding only; false: the sequence has no such
// tile.
__device__ __forceinline__ bool pg_range(const PgArgs& a, const PgSeq& s, int tile, int kR, int& lo, int& hi) {
  if (tile < 0 || (int64_t)tile * kR >= (int64_t)s.span * a.Hg) return false;
  lo = s.lo;
  hi = s.hi;
  const int first = (tile * kR) / a.Hg, last = min(((tile + 1) * kR - 1) / a.Hg, s.len - 1);
  if (first >= s.len) hi = lo;
  else if (a.causal) hi = max(min(hi, s.n - s.len + last + 1), 0);
  if (a.win >= 0) lo = max(lo, (max(s.n - s.len + first, 0) - a.win) & ~(kPgTile - 1));
  lo = min(lo, hi);
  return true;
}

// A tile and all its keys for each workgroup.  Group fastest, so that the workgroups of an XCD (every eighth) read few
// groups' caches; the causal rows with the most keys first.
template <class W>
__global__ __launch_bounds__(W::kThreads) void pg_direct_kernel(PgArgs a) {
  extern __shared__ __align__(16) uint8_t lds[];
  const int rank = blockIdx.x / a.G, kvg = blockIdx.x - rank * a.G;
  const int slot = a.slots - 1 - rank;
  const int b = pg_find(a, a.cu_q, slot, W::kR);
  const PgSeq s = pg_seq(a, b);
  const int tile = slot - pg_slot(s.start, a.Hg, b, W::kR);
  int lo, hi;
  if (!pg_range(a, s, tile, W::kR, lo, hi)) return;
  W::item(a, s, b, tile, kvg, lo, hi, true, nullptr, lds);
}

// The line of units: slot x takes [at[x], at[x + 1]) of each group, a tile's first kExtra for what it costs beside
// its keys (start and end, three units' time in either way).  Every workgroup of the split kernel makes it alike, in
// LDS; the first writes it out for the join.
constexpr int kPgExtra = 3;
constexpr int kPgLineCu = 1024;
struct PgLine {
  int at[kPgMaxSlots + 1];
  uint16_t seq[kPgMaxSlots];
  int32_t cu[kPgLineCu];
};

template <class W>
__device__ __forceinline__ void pg_line(const PgArgs& a, PgLine& line, int threads) {
  const int tid = threadIdx.x;
  const bool copy = a.cu_q && a.B <= kPgLineCu;
  if (copy)
    for (int b = tid; b < a.B; b += threads) line.cu[b] = a.cu_q[b];
  __syncthreads();
  for (int x = tid; x < a.slots; x += threads) {
    const int b = pg_find(a, copy ? line.cu : a.cu_q, x, W::kR);
    const PgSeq s = pg_seq(a, b);
    int lo, hi, units = 0;
    // A tile without keys takes a unit too: it writes its zeros.
    if (pg_range(a, s, x - pg_slot(s.start, a.Hg, b, W::kR), W::kR, lo, hi))
      units = kPgExtra + max(1, (hi - lo + W::kUnitKeys - 1) / W::kUnitKeys);
    line.seq[x] = (uint16_t)b;
    line.at[x + 1] = units;
  }
  if (tid == 0) line.at[0] = 0;
  __syncthreads();
  if (tid < kWave) {
    int sum = 0;
    for (int x = tid; x < ((a.slots + kWave - 1) & ~(kWave - 1)); x += kWave) {
      int v = x < a.slots ? line.at[x + 1] : 0;
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) {
        const int u = __shfl_up(v, o, kWave);
        if (tid >= o) v += u;
      }
      if (x < a.slots) line.at[x + 1] = sum + v;
      sum += __shfl(v, kWave - 1, kWave);
    }
  }
  __syncthreads();
}

// Units of a workgroup's part of the line.
__device__ __forceinline__ int pg_share(const PgArgs& a, int total) { return max((total + a.wgs - 1) / a.wgs, 1); }

// A workgroup has at most two tiles that others share: one begun before its part of the line, and one that goes on
// behind it.
template <class W>
__device__ __forceinline__ float* pg_part(const PgArgs& a, int wg, bool begun_before) {
  return a.part + (int64_t)(2 * wg + (begun_before ? 0 : 1)) * pg_part_floats<W::kR, W::kD>();
}

template <class W>
__global__ __launch_bounds__(W::kThreads) void pg_split_kernel(PgArgs a) {
  extern __shared__ __align__(16) uint8_t lds[];
  PgLine& line = *reinterpret_cast<PgLine*>(lds + W::kLds);
  pg_line<W>(a, line, W::kThreads);
  if (blockIdx.x == 0) {
    for (int x = threadIdx.x; x <= a.slots; x += W::kThreads) {
      a.line[x] = line.at[x];
      if (x < a.slots) a.line[a.slots + 1 + x] = line.seq[x];
    }
  }
  const int total = line.at[a.slots] * a.G, share = pg_share(a, total);
  const int begin = min((int)min((int64_t)blockIdx.x * share, (int64_t)total), total);
  const int end = (int)min((int64_t)begin + share, (int64_t)total);
  int x = 0;  // the last slot whose line starts at or before `begin`
  {
    int x1 = a.slots - 1;
    while (x < x1) {
      const int mid = (x + x1 + 1) >> 1;
      if (line.at[mid] * a.G <= begin) x = mid;
      else x1 = mid - 1;
    }
  }
  x = __builtin_amdgcn_readfirstlane(x);
  for (; x < a.slots; ++x) {
    const int from = __builtin_amdgcn_readfirstlane(line.at[x]) * a.G;
    if (from >= end) break;
    const int length = __builtin_amdgcn_readfirstlane(line.at[x + 1] - line.at[x]);
    if (length == 0) continue;
    const int b = __builtin_amdgcn_readfirstlane((int)line.seq[x]);
    const PgSeq s = pg_seq(a, b);
    const int tile = x - pg_slot(s.start, a.Hg, b, W::kR);
    int lo, hi;
    if (!pg_range(a, s, tile, W::kR, lo, hi)) break;  // not reached: the slot has units
    for (int kvg = max(0, (begin - from) / length); kvg < a.G; ++kvg) {
      const int u0 = from + kvg * length + kPgExtra, u1 = u0 + length - kPgExtra;  // the tile's units on the line
      if (u0 - kPgExtra >= end) break;
      const int c0 = max(u0, begin), c1 = min(u1, end);
      if (c0 >= c1) continue;
      const int k0 = (int)min((int64_t)hi, lo + (int64_t)(c0 - u0) * W::kUnitKeys);
      const int k1 = (int)min((int64_t)hi, lo + (int64_t)(c1 - u0) * W::kUnitKeys);
      W::item(a, s, b, tile, kvg, k0, k1, c0 == u0 && c1 == u1, pg_part<W>(a, blockIdx.x, u0 < begin), lds);
    }
  }
}

// Joins the parts of each tile whose units lie in more than one workgroup's share: workgroup = (slot and group, rows).
// kGroups groups of threads take every kGroups-th part of a pass's rows, 8 columns a thread, and are summed through
// LDS: four for the tiles of few rows, whose keys may lie in many parts, one for those of 256, which have many rows.
// Those have a workgroup a pass as long as the slots are few (64 queries of 64 heads over 30000 keys: 16 parts a tile,
// 21.7 us with four passes a workgroup, 8.8 with one), and four passes a workgroup where most slots may hold no tile
// (800 sequences of 5 tokens: 79.7 us with one pass, 21.1 with four).
template <class W>
struct PgJoin {
  static constexpr int kPerRow = W::kD / 8;
  static constexpr int kGroups = W::kR == kPrRows ? 1 : 4;
  static constexpr int kPass = kPgThreads / kGroups / kPerRow;  // rows of a pass
  static constexpr int kMost = W::kR == kPrRows ? 4 : 1;        // passes of a workgroup
  static_assert(W::kR % (kMost * kPass) == 0, "whole groups of rows");
};
template <class W>
__global__ __launch_bounds__(kPgThreads) void pg_join_kernel(PgArgs a) {
  typedef PgJoin<W> J;
  constexpr int kR = W::kR, kD = W::kD;
  constexpr bool kF16 = W::kF16;
  const int x = blockIdx.x / a.G, kvg = blockIdx.x - x * a.G;
  const int from = a.line[x], length = a.line[x + 1] - from, share = pg_share(a, a.line[a.slots] * a.G);
  const int b = a.line[a.slots + 1 + x];
  if (length == 0) return;
  const int u0 = from * a.G + kvg * length + kPgExtra, u1 = u0 + length - kPgExtra;
  const int w0 = u0 / share, np = (u1 - 1) / share - w0 + 1;
  if (np == 1) return;
  const PgSeq s = pg_seq(a, b);
  const int tile = x - pg_slot(s.start, a.Hg, b, kR);
  const int group = threadIdx.x / (kPgThreads / J::kGroups), in = threadIdx.x % (kPgThreads / J::kGroups);
  const int t = in % J::kPerRow, c0 = 8 * t;
  const auto part = [&](int p) { return pg_part<W>(a, w0 + p, u0 < (w0 + p) * share); };
  __shared__ float sums[J::kGroups][9][kPgThreads / J::kGroups];
  const int rows = kR / gridDim.y;  // of the workgroup
  for (int r0 = 0; r0 < rows; r0 += J::kPass) {
    const int hh = blockIdx.y * rows + r0 + in / J::kPerRow;
    const int rho = tile * kR + hh;
    if (rho - in / J::kPerRow >= s.span * a.Hg) break;  // no row of the pass
    const bool live = rho < s.span * a.Hg;
    float M = -kPgInf;
    for (int p = t; p < np; p += J::kPerRow) M = fmaxf(M, part(p)[kR * kD + 2 * hh]);
#pragma unroll
    for (int o = 1; o < J::kPerRow; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, kWave));
    const int i = rho / a.Hg, h = kvg * a.Hg + rho - i * a.Hg;
    const float M_use = M == -kPgInf ? 0.f : M, sink = live ? pg_sink(a, h) : -kPgInf;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = 0.f;
    constexpr int kAhead = J::kGroups == 1 ? 4 : 8;  // parts whose loads are in flight together
    for (int p0 = group; p0 < np; p0 += J::kGroups * kAhead) {
      f32x4 x0[kAhead], x1[kAhead];
      float m[kAhead], l[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const float* pp = part(min(p0 + J::kGroups * j, np - 1));
        x0[j] = *reinterpret_cast<const f32x4*>(pp + hh * kD + c0);
        x1[j] = *reinterpret_cast<const f32x4*>(pp + hh * kD + c0 + 4);
        m[j] = pp[kR * kD + 2 * hh];
        l[j] = pp[kR * kD + 2 * hh + 1];
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const float f = p0 + J::kGroups * j < np ? fast_exp2(m[j] - M_use) : 0.f;
        sum += f * l[j];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          acc[k] += f * x0[j][k];
          acc[4 + k] += f * x1[j][k];
        }
      }
    }
    if constexpr (J::kGroups > 1) {
#pragma unroll
      for (int k = 0; k < 8; ++k) sums[group][k][in] = acc[k];
      sums[group][8][in] = sum;
      __syncthreads();
      if (group > 0) return;  // one pass
      sum = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] = 0.f;
#pragma unroll
      for (int w = 0; w < J::kGroups; ++w) {
        sum += sums[w][8][in];
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] += sums[w][k][in];
      }
    }
    if (!live) continue;
    const PgEnd e = pg_end(M, sum, sink);
    const float inv = e.scale;
    const int64_t orow = (int64_t)(s.start + i) * a.H + h;
    *reinterpret_cast<u32x4*>(a.out + orow * kD + c0) =
        u32x4{gqa_pack<kF16>(acc[0] * inv, acc[1] * inv), gqa_pack<kF16>(acc[2] * inv, acc[3] * inv),
              gqa_pack<kF16>(acc[4] * inv, acc[5] * inv), gqa_pack<kF16>(acc[6] * inv, acc[7] * inv)};
    if (c0 == 0) a.lse[orow] = e.lse;
  }
}

// The launch of a call, from sizes that the host knows: T tokens, B sequences, at most `most` keys each.
struct PgPlan {
  int rows;       // of a tile: 16, 32 (pg_keys) or 256 (pg_rows)
  int64_t slots;  // tiles at most, in each group
  int wgs;        // workgroups that share the line of units; 0: a tile each
};

static PgPlan pg_plan(int64_t T, int64_t B, int64_t H, int64_t G, int64_t most) {
  PgPlan p;
  const int64_t Hg = H / G;
  p.rows = T * Hg <= 16 * B ? 16 : T * Hg <= 32 * B ? 32 : kPrRows;
  p.slots = T * Hg / p.rows + B + 1;
  p.wgs = 0;
  // One workgroup fits a CU.  Fewer than two rounds of tiles share the line, and batches of many sequences, where slots
  // without a tile lie between the others (a workgroup each for 64 x 8192 keys put the tiles on every other XCD: 330 us
  // instead of 199).
  const int64_t unit = p.rows == kPrRows ? kPrTile : kPgUnit;
  const int64_t units = p.slots * G * ((most + unit - 1) / unit + 1 + kPgExtra);
  if (p.slots <= kPgMaxSlots && units < ((int64_t)1 << 30) && (p.slots * G < 512 || 4 * (B + 1) > p.slots))
    p.wgs = (int)(units < 256 ? units : 256);
  return p;
}

// The largest grid, of tiles in each group, within the 2^32 threads of a launch (the shared line's and the join's are
// smaller).  T * H < 2^31, B, G <= 65535.
bool paged_gqa_fits(int64_t T, int64_t B, int64_t H, int64_t G, int64_t most) {
  const PgPlan p = pg_plan(T, B, H, G, most);
  return p.slots * G < ((int64_t)1 << 32) / (p.rows == kPrRows ? kPrThreads : kPgThreads);
}

static size_t pg_part_bytes(const PgPlan& p, int64_t D) { return (size_t)(2 * p.wgs) * p.rows * (D + 2) * sizeof(float); }

size_t paged_gqa_workspace_bytes(int64_t T, int64_t B, int64_t H, int64_t G, int64_t D, int64_t most) {
  const PgPlan p = pg_plan(T, B, H, G, most);
  if (p.wgs == 0) return 0;
  return pg_part_bytes(p, D) + (size_t)(2 * p.slots + 1) * sizeof(int32_t);
}

template <class W>
static hipError_t pg_launch(const PgArgs& a, hipStream_t stream) {
  constexpr int split_lds = W::kLds + (int)sizeof(PgLine);
  static_assert(W::kLds % 16 == 0 && split_lds <= 160 * 1024, "LDS");
  const dim3 tiles((unsigned)((int64_t)a.slots * a.G));
  hipError_t e;
  if (a.wgs == 0) {
    e = set_dynamic_lds_once<pg_direct_kernel<W>>(W::kLds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((pg_direct_kernel<W>), tiles, dim3(W::kThreads), W::kLds, stream, a);
    return hipGetLastError();
  }
  e = set_dynamic_lds_once<pg_split_kernel<W>>(split_lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((pg_split_kernel<W>), dim3(a.wgs), dim3(W::kThreads), split_lds, stream, a);
  typedef PgJoin<W> J;
  const dim3 join(tiles.x, W::kR / J::kPass / (tiles.x > kPgFewSlots ? J::kMost : 1));
  hipLaunchKernelGGL((pg_join_kernel<W>), join, dim3(kPgThreads), 0, stream, a);
  return hipGetLastError();
}

template <bool kF16, int kD>
static hipError_t pg_dispatch(const PgArgs& a, int rows, hipStream_t stream) {
  if (rows == kPrRows && a.block_size % 8 == 0) return pg_launch<PgRows<kF16, kD, true>>(a, stream);
  if (rows == kPrRows) return pg_launch<PgRows<kF16, kD, false>>(a, stream);
  return rows == 32 ? pg_launch<PgKeys<kF16, kD, 2>>(a, stream) : pg_launch<PgKeys<kF16, kD, 1>>(a, stream);
}

// Caller validated: D in {64, 128}, H a multiple of G, T * H < 2^31 - 65536, pool rows < 2^31,
// max_blocks * block_size <= 2^31 - 1 - 4096, paged_gqa_fits, sm_scale > 0, the workspace as
// paged_gqa_workspace_bytes says.
hipError_t launch_paged_gqa(int is_fp16, const void* q, const void* kc, const void* vc, const int32_t* table,
                            const int32_t* cu_q, const int32_t* q_len, const int32_t* kv_len, int64_t T, int64_t B,
                            int64_t S, int64_t H, int64_t G, int64_t D, int64_t num_blocks, int64_t block_size,
                            int64_t max_blocks, int causal, int64_t win_left, const float* sinks, float sm_scale,
                            void* out, float* lse, void* workspace, hipStream_t stream) {
  if (T == 0 || H == 0) return hipSuccess;
  const PgPlan p = pg_plan(T, B, H, G, max_blocks * block_size);
  PgArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.kc = static_cast<const uint16_t*>(kc);
  a.vc = static_cast<const uint16_t*>(vc);
  a.table = table;
  a.cu_q = cu_q;
  a.q_len = q_len;
  a.kv_len = kv_len;
  a.sinks = sinks;
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.part = static_cast<float*>(workspace);
  a.line = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + pg_part_bytes(p, D));
  a.T = (int)T;
  a.B = (int)B;
  a.S = (int)S;
  a.H = (int)H;
  a.G = (int)G;
  a.Hg = (int)(H / G);
  a.block_size = (int)block_size;
  a.max_blocks = (int)max_blocks;
  a.num_blocks = (int)num_blocks;
  a.causal = causal;
  a.win = win_left < max_blocks * block_size ? (int)win_left : -1;  // a window as long as the cache is none
  a.wgs = p.wgs;
  a.slots = (int)p.slots;
  a.div_mul = 0;
  a.div_shift = 0;
  if (block_size > 1) {
    int l = 0;
    while (((int64_t)1 << l) < block_size) ++l;
    a.div_mul = (uint32_t)((((uint64_t)1 << (31 + l)) / (uint64_t)block_size) + 1);
    a.div_shift = l - 1;
  }
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  if (D == 128) return is_fp16 ? pg_dispatch<true, 128>(a, p.rows, stream) : pg_dispatch<false, 128>(a, p.rows, stream);
  return is_fp16 ? pg_dispatch<true, 64>(a, p.rows, stream) : pg_dispatch<false, 64>(a, p.rows, stream);
}

}  // namespace dsa
