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
// cut into tiles of 16 kHB rows, so that each key is read once for a tile whatever Hg.  Tile i of sequence b has
// the slot floor(start_b * Hg / rows) + b + i: sequences get disjoint slots without a prefix sum, and a grid of
// floor(T * Hg / rows) + B + 1 slots holds them all (b = B is the padding behind the last packed sequence).
//
// Work split.  A workgroup's four waves take 32 keys each of a unit of 128, every wave with a ring of its own
// in LDS (no workgroup barrier in the loop), an online softmax and a merge at the end.  Where there are tiles enough
// a workgroup takes a tile and all its keys.  Otherwise the units of all tiles form one line that is cut into
// equal parts, a workgroup each, so that batches of uneven lengths load the card evenly; a tile whose line is
// cut leaves parts (unnormalised sums in fp32, with maximum and sum) that a second launch joins.
//
// Per 32 keys and wave: S^T = K Q^T (keys on the M axis of 16x16x32 products), the softmax in base 2 (a lane holds
// 8 scores of one row), O^T += V^T P^T with V^T through transposing LDS reads.
#include "gqa_common.hpp"

namespace dsa {

constexpr int kPgTile = 32;                 // keys a wave takes at once
constexpr int kPgWaves = 4;
constexpr int kPgThreads = kPgWaves * kWave;
constexpr int kPgUnit = kPgWaves * kPgTile;  // 128 keys
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
  float* part;            // parts: sums [16 kHB, D], then (maximum, sum) [16 kHB, 2]
  int T, B, S, H, G, Hg, block_size, max_blocks, num_blocks, causal, win, wgs;
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

template <int kHB, int kD>
__host__ __device__ constexpr int pg_part_floats() { return 16 * kHB * (kD + 2); }

// Two stages of K and V of 32 keys a wave; the merge reuses a wave's ring, its (maximum, sum) lie behind.
template <int kHB, int kD>
__host__ __device__ constexpr int pg_lds_bytes() { return kPgWaves * 2 * 2 * kPgTile * kD * 2 + kPgWaves * 16 * kHB * 2 * 4; }

// Keys behind a sequence's last one, and of pages outside the pool, load this row: 0 times what lies there need
// not be 0.
static __device__ __align__(128) uint8_t kPgZeroRow[256];

// The keys [k0, k1) of tile `tile` of sequence s, group kvg; `whole`: these are all its keys (the result goes to
// out and lse, otherwise to the part).
template <bool kF16, int kD, int kHB>
__device__ __forceinline__ void pg_item(const PgArgs& a, const PgSeq& s, int b, int tile, int kvg, int k0, int k1,
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
      const int blk = j / a.block_size, page = bt[blk];
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
    if (ok_cur != 0xffffffffu || j0 + kPgTile - 1 > all_lim || j0 < all_low) {
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
  constexpr float kLn2 = 0.6931471805599453f;
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
      float M2 = M_use, f = 1.f;
      if (a.sinks) {
        const float sk = a.sinks[h] * 1.4426950408889634f;
        M2 = fmaxf(M, sk);
        M2 = M2 == -kPgInf ? 0.f : M2;
        f = fast_exp2(M - M2);
        sum = sum * f + fast_exp2(sk - M2);
      }
      const float inv = sum > 0.f ? f / sum : 0.f;
      *reinterpret_cast<u32x4*>(a.out + orow * kD + c0) =
          u32x4{gqa_pack<kF16>(acc[0] * inv, acc[1] * inv), gqa_pack<kF16>(acc[2] * inv, acc[3] * inv),
                gqa_pack<kF16>(acc[4] * inv, acc[5] * inv), gqa_pack<kF16>(acc[6] * inv, acc[7] * inv)};
      if (c0 == 0) a.lse[orow] = sum > 0.f ? (M2 + fast_log2(sum)) * kLn2 : -kPgInf;
    }
  }
  __syncthreads();  // the rings are free for the next item
}

// Slot of the first tile of sequence b, rows of one tile kR: strictly increasing in b.
__device__ __forceinline__ int pg_slot(int start, int Hg, int b, int kR) {
  return (int)((int64_t)start * Hg / kR) + b;
}
__device__ __forceinline__ int pg_start(const PgArgs& a, int b) {
  if (!a.cu_q) return min(b, a.B) * a.S;
  return b > 0 ? min(max(a.cu_q[b - 1], 0), a.T) : 0;
}

// A tile and all its keys for each workgroup: blockIdx.x = slot, blockIdx.y = group.
template <bool kF16, int kD, int kHB>
__global__ __launch_bounds__(kPgThreads) void pg_direct_kernel(PgArgs a) {
  extern __shared__ __align__(16) uint8_t lds[];
  constexpr int kR = 16 * kHB;
  // The causal rows with the most keys first.
  const int slot = (int)(gridDim.x - 1 - blockIdx.x);
  int b0 = 0, b1 = a.B;  // the last b whose first slot is not past ours
  while (b0 < b1) {
    const int mid = (b0 + b1 + 1) >> 1;
    if (pg_slot(pg_start(a, mid), a.Hg, mid, kR) <= slot) b0 = mid;
    else b1 = mid - 1;
  }
  const PgSeq s = pg_seq(a, b0);
  const int tile = slot - pg_slot(s.start, a.Hg, b0, kR);
  if (tile < 0 || (int64_t)tile * kR >= (int64_t)s.span * a.Hg) return;
  int lo = s.lo, hi = s.hi;
  const int first = (tile * kR) / a.Hg, last = min(((tile + 1) * kR - 1) / a.Hg, s.span - 1);
  if (a.causal) hi = max(min(hi, s.n - s.len + last + 1), 0);
  if (a.win >= 0) lo = max(lo, (max(s.n - s.len + first, 0) - a.win) & ~(kPgTile - 1));
  pg_item<kF16, kD, kHB>(a, s, b0, tile, (int)blockIdx.y, min(lo, hi), hi, true, nullptr, lds);
}

// Units (128 keys) of each tile of the sequence, at least one: a tile without keys writes its zeros.
__device__ __forceinline__ int pg_units(const PgSeq& s) { return max(1, (s.hi - s.lo + kPgUnit - 1) / kPgUnit); }
__device__ __forceinline__ int pg_tiles(const PgArgs& a, const PgSeq& s, int kR) {
  return (int)(((int64_t)s.span * a.Hg + kR - 1) / kR);
}

// The line of units, shared by the split kernel and the join: thread t sums sequences [t * per, (t + 1) * per).
// Returns the thread's exclusive prefix; `total` is the line's length.
__device__ __forceinline__ int64_t pg_line(const PgArgs& a, int kR, int64_t& total, int64_t* scratch) {
  const int per = (a.B + 1 + kPgThreads - 1) / kPgThreads;
  const int b0 = threadIdx.x * per;
  int64_t sum = 0;
  for (int i = 0; i < per; ++i) {
    if (b0 + i > a.B) break;
    const PgSeq s = pg_seq(a, b0 + i);
    sum += (int64_t)pg_tiles(a, s, kR) * a.G * pg_units(s);
  }
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  int64_t incl = sum;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int64_t v = __shfl_up(incl, o, kWave);
    if (lane >= o) incl += v;
  }
  if (lane == kWave - 1) scratch[wave] = incl;
  __syncthreads();
  int64_t base = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPgWaves; ++w) {
    if (w < wave) base += scratch[w];
    total += scratch[w];
  }
  __syncthreads();
  return base + incl - sum;
}

// Units of a workgroup's part of the line.
__device__ __forceinline__ int64_t pg_share(int64_t total, int wgs) { return max((total + wgs - 1) / wgs, (int64_t)1); }

template <bool kF16, int kD, int kHB>
__global__ __launch_bounds__(kPgThreads) void pg_split_kernel(PgArgs a) {
  extern __shared__ __align__(16) uint8_t lds[];
  constexpr int kR = 16 * kHB;
  int64_t* scratch = reinterpret_cast<int64_t*>(lds);
  int64_t total;
  const int64_t before = pg_line(a, kR, total, scratch);
  const int64_t share = pg_share(total, a.wgs);
  int64_t u = (int64_t)blockIdx.x * share;
  const int64_t end = min(u + share, total);
  if (u >= end) return;
  // The sequence that unit u lies in, and the line's units before it.
  {
    const int per = (a.B + 1 + kPgThreads - 1) / kPgThreads;
    int64_t at = before;
    for (int i = 0; i < per; ++i) {
      const int b = threadIdx.x * per + i;
      if (b > a.B) break;
      const PgSeq s = pg_seq(a, b);
      const int64_t len = (int64_t)pg_tiles(a, s, kR) * a.G * pg_units(s);
      if (u >= at && u < at + len) {
        scratch[8] = at;
        scratch[9] = b;
      }
      at += len;
    }
  }
  __syncthreads();
  int64_t at = scratch[8];
  int b = (int)scratch[9];
  __syncthreads();
  at = ((int64_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
  b = __builtin_amdgcn_readfirstlane(b);
  while (u < end) {
    const PgSeq s = pg_seq(a, b);
    const int units = pg_units(s);
    const int64_t items = (int64_t)pg_tiles(a, s, kR) * a.G;
    while (u < end && u < at + items * units) {
      const int item = (int)((u - at) / units);
      const int64_t u0 = at + (int64_t)item * units;  // the item's units on the line: [u0, u0 + units)
      const int64_t stop = min(end, u0 + units);
      const bool whole = u == u0 && stop == u0 + units;
      const int tile = item / a.G, kvg = item - tile * a.G;
      const int k0 = s.lo + (int)(u - u0) * kPgUnit;
      const int k1 = (int)min((int64_t)s.hi, s.lo + (stop - u0) * kPgUnit);
      const int64_t id = (int64_t)(pg_slot(s.start, a.Hg, b, kR) + tile) * a.G + kvg;
      pg_item<kF16, kD, kHB>(a, s, b, tile, kvg, min(k0, k1), k1, whole,
                             whole ? nullptr : a.part + (id + blockIdx.x) * pg_part_floats<kHB, kD>(), lds);
      u = stop;
    }
    at += items * units;
    ++b;
  }
}

// Joins the parts of each tile whose units lie in more than one workgroup's share: workgroup = (slot, group).
template <bool kF16, int kD, int kHB>
__global__ __launch_bounds__(kPgThreads) void pg_join_kernel(PgArgs a) {
  constexpr int kR = 16 * kHB;
  __shared__ int64_t scratch[16];
  int64_t total;
  const int64_t before = pg_line(a, kR, total, scratch);
  const int64_t share = pg_share(total, a.wgs);
  const int slot = blockIdx.x, kvg = blockIdx.y;
  if (threadIdx.x == 0) scratch[9] = -1;
  __syncthreads();
  {
    const int per = (a.B + 1 + kPgThreads - 1) / kPgThreads;
    int64_t at = before;
    for (int i = 0; i < per; ++i) {
      const int b = threadIdx.x * per + i;
      if (b > a.B) break;
      const PgSeq s = pg_seq(a, b);
      const int tiles = pg_tiles(a, s, kR), first = pg_slot(s.start, a.Hg, b, kR);
      if (slot >= first && slot < first + tiles) {
        scratch[8] = at;
        scratch[9] = b;
      }
      at += (int64_t)tiles * a.G * pg_units(s);
    }
  }
  __syncthreads();
  const int b = (int)scratch[9];
  if (b < 0) return;
  const PgSeq s = pg_seq(a, b);
  const int units = pg_units(s), tile = slot - pg_slot(s.start, a.Hg, b, kR);
  const int64_t u0 = scratch[8] + ((int64_t)tile * a.G + kvg) * units;
  const int w0 = (int)(u0 / share), w1 = (int)((u0 + units - 1) / share);
  if (w0 == w1) return;
  const int64_t id = (int64_t)slot * a.G + kvg;
  const float* base = a.part + (id + w0) * pg_part_floats<kHB, kD>();
  constexpr int kPerRow = kD / 8;
  constexpr int kRowsPass = kPgThreads / kPerRow;
  constexpr float kLn2 = 0.6931471805599453f;
  const int rows = s.span * a.Hg;
#pragma unroll
  for (int r0 = 0; r0 < kR; r0 += kRowsPass) {
    const int hh = r0 + threadIdx.x / kPerRow, c0 = 8 * (threadIdx.x % kPerRow);
    const int rho = tile * kR + hh;
    if (hh >= kR || rho >= rows) continue;
    const int i = rho / a.Hg, h = kvg * a.Hg + rho - i * a.Hg;
    const int np = w1 - w0 + 1;
    float M = -kPgInf;
    for (int p = 0; p < np; ++p) M = fmaxf(M, base[(int64_t)p * pg_part_floats<kHB, kD>() + kR * kD + 2 * hh]);
    const float sk = a.sinks ? a.sinks[h] * 1.4426950408889634f : -kPgInf;
    M = fmaxf(M, sk);
    const float M_use = M == -kPgInf ? 0.f : M;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = fast_exp2(sk - M_use);
    for (int p = 0; p < np; ++p) {
      const float* pp = base + (int64_t)p * pg_part_floats<kHB, kD>();
      const float f = fast_exp2(pp[kR * kD + 2 * hh] - M_use);
      sum += f * pp[kR * kD + 2 * hh + 1];
      const f32x4 x0 = *reinterpret_cast<const f32x4*>(pp + hh * kD + c0);
      const f32x4 x1 = *reinterpret_cast<const f32x4*>(pp + hh * kD + c0 + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        acc[k] += f * x0[k];
        acc[4 + k] += f * x1[k];
      }
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    const int64_t orow = (int64_t)(s.start + i) * a.H + h;
    *reinterpret_cast<u32x4*>(a.out + orow * kD + c0) =
        u32x4{gqa_pack<kF16>(acc[0] * inv, acc[1] * inv), gqa_pack<kF16>(acc[2] * inv, acc[3] * inv),
              gqa_pack<kF16>(acc[4] * inv, acc[5] * inv), gqa_pack<kF16>(acc[6] * inv, acc[7] * inv)};
    if (c0 == 0) a.lse[orow] = sum > 0.f ? (M_use + fast_log2(sum)) * kLn2 : -kPgInf;
  }
}

// The launch of a call, from sizes that the host knows: T tokens, B sequences, at most `most` keys each.
struct PgPlan {
  int hb;         // 16-row blocks of a tile
  int64_t slots;  // tiles at most, in each group
  int wgs;        // workgroups that share the line of units; 0: a tile each
};

static PgPlan pg_plan(int64_t T, int64_t B, int64_t H, int64_t G, int64_t most) {
  PgPlan p;
  const int64_t Hg = H / G;
  p.hb = T * Hg > 16 * B ? 2 : 1;
  p.slots = T * Hg / (16 * p.hb) + B + 1;
  p.wgs = 0;
  if (p.slots * G < 1024) {
    const int64_t units = p.slots * G * ((most + kPgUnit - 1) / kPgUnit + 1);
    p.wgs = (int)(units < 256 ? units : 256);
  }
  return p;
}

static int pg_floats(int hb, int64_t D) { return 16 * hb * ((int)D + 2); }

size_t paged_gqa_workspace_bytes(int64_t T, int64_t B, int64_t H, int64_t G, int64_t D, int64_t most) {
  const PgPlan p = pg_plan(T, B, H, G, most);
  if (p.wgs == 0) return 0;
  return (size_t)(p.slots * G + p.wgs) * pg_floats(p.hb, D) * sizeof(float);
}

template <bool kF16, int kD, int kHB>
static hipError_t pg_launch(PgArgs& a, const PgPlan& p, hipStream_t stream) {
  constexpr int lds = pg_lds_bytes<kHB, kD>();
  static_assert(lds <= 160 * 1024 && 16 * kHB * kD * 4 <= 4 * kPgTile * kD * 2, "a wave's sums fit its ring");
  const dim3 tiles((unsigned)p.slots, (unsigned)a.G);
  hipError_t e;
  if (p.wgs == 0) {
    e = set_dynamic_lds_once<pg_direct_kernel<kF16, kD, kHB>>(lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((pg_direct_kernel<kF16, kD, kHB>), tiles, dim3(kPgThreads), lds, stream, a);
    return hipGetLastError();
  }
  e = set_dynamic_lds_once<pg_split_kernel<kF16, kD, kHB>>(lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((pg_split_kernel<kF16, kD, kHB>), dim3(p.wgs), dim3(kPgThreads), lds, stream, a);
  hipLaunchKernelGGL((pg_join_kernel<kF16, kD, kHB>), tiles, dim3(kPgThreads), 0, stream, a);
  return hipGetLastError();
}

template <bool kF16, int kD>
static hipError_t pg_dispatch(PgArgs& a, const PgPlan& p, hipStream_t stream) {
  return p.hb == 2 ? pg_launch<kF16, kD, 2>(a, p, stream) : pg_launch<kF16, kD, 1>(a, p, stream);
}

// Caller validated: D in {64, 128}, H a multiple of G, T * H < 2^31, G <= 65535, pool rows < 2^31,
// max_blocks * block_size <= 2^31 - 1 - 1024, sm_scale > 0, the workspace as paged_gqa_workspace_bytes says.
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
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  if (D == 128) return is_fp16 ? pg_dispatch<true, 128>(a, p, stream) : pg_dispatch<false, 128>(a, p, stream);
  return is_fp16 ? pg_dispatch<true, 64>(a, p, stream) : pg_dispatch<false, 64>(a, p, stream);
}

}  // namespace dsa
