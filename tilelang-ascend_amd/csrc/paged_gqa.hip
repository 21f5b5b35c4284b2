// Attention of new tokens over a paged cache: the launch.  The kernels, the mathematics and the rules that choose among
// them stand in paged_gqa_kernels.hpp.
#include "paged_gqa_kernels.hpp"

namespace dsa {

bool paged_gqa_fits(int64_t T, int64_t B, int64_t H, int64_t G, int64_t most) {
  return pg_fits(pg_plan(T, B, H, G, most, false), G);
}

size_t paged_gqa_workspace_bytes(int64_t T, int64_t B, int64_t H, int64_t G, int64_t D, int64_t most) {
  return pg_workspace_bytes(pg_plan(T, B, H, G, most, false), D);
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
  const PgPlan p = pg_plan(T, B, H, G, max_blocks * block_size, false);
  PgArgs a = pg_args({T, B, S, H, G, D, num_blocks, block_size, max_blocks}, q, kc, vc, table, cu_q, q_len, kv_len,
                     win_left, sinks, sm_scale, out, lse, workspace, p);
  a.causal = causal;
  if (D == 128)
    return is_fp16 ? pg_dispatch<true, 128, false>(a, p.rows, stream) : pg_dispatch<false, 128, false>(a, p.rows, stream);
  return is_fp16 ? pg_dispatch<true, 64, false>(a, p.rows, stream) : pg_dispatch<false, 64, false>(a, p.rows, stream);
}

}  // namespace dsa
