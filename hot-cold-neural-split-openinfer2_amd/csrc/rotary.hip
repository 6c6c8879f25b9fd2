// Rotary positions of q and k, each token at its own position.
//
// Bound by the bytes of q and k, in and out, from some thousand tokens on; a
// step of 16 tokens (4.2 us) by its launch and one chain of loads, turns and
// stores.
#include "rotary.h"

#include "capi_util.h"

namespace oi2 {
namespace {

template <bool BF16, bool WIDE>
__global__ __launch_bounds__(256) void k_rotary(RotaryArgs a) {
  rotate_tokens<BF16, WIDE, 256>(a, blockIdx.x);
}

}  // namespace

int check_rotary(const oi2_rotary* r) {
  OI2_CHECK_ARG(r && r->freq && (uintptr_t)r->freq % 8 == 0, "rotary frequencies must be non-null and 8-byte aligned");
  OI2_CHECK_ARG(r->head_dim >= 2 && r->head_dim <= 256 && r->head_dim % 2 == 0, "head_dim %d: even, 2 to 256", r->head_dim);
  OI2_CHECK_ARG(r->rotary_dim >= 2 && r->rotary_dim <= r->head_dim && r->rotary_dim % 2 == 0,
                "rotary_dim %d: even, 2 to head_dim %d", r->rotary_dim, r->head_dim);
  return OI2_OK;
}

}  // namespace oi2

using namespace oi2;

extern "C" int oi2_rotary_apply(const oi2_rotary* r, int32_t dtype, int32_t n_tokens, const int32_t* positions,
                                const oi2_heads* q, void* q_out, const oi2_heads* k, void* k_out, void* stream) {
  clear_error();
  if (int rc = check_rotary(r)) return rc;
  const bool zero = dtype & OI2_ZERO_LEFT_OUT;
  dtype &= ~OI2_ZERO_LEFT_OUT;
  OI2_CHECK_ARG(dtype == OI2_DTYPE_F16 || dtype == OI2_DTYPE_BF16, "dtype %d: fp16 or bf16", dtype);
  OI2_CHECK_ARG(n_tokens >= 0, "%d tokens", n_tokens);
  OI2_CHECK_ARG(q && k && q->heads >= 0 && k->heads >= 0 && q->heads <= 1 << 16 && k->heads <= 1 << 16, "null q or k, or heads out of range");
  if (n_tokens == 0 || q->heads + k->heads == 0) return OI2_OK;
  OI2_CHECK_ARG((!q->heads || (q->data && q_out)) && (!k->heads || (k->data && k_out)), "null q or k data");
  OI2_CHECK_ARG(positions, "null positions");
  RotaryArgs a{};
  rotary_describe(a, r, n_tokens, positions, zero);
  const bool wide = rotary_fill(a, q, q_out, k, k_out);
  for (int w = 0; w < 2; ++w)
    OI2_CHECK_ARG(!a.heads[w] || ((uintptr_t)a.src[w] % 2 == 0 && (uintptr_t)a.dst[w] % 2 == 0), "q and k must be 2-byte aligned");
  const int64_t groups = rotary_workgroups(a);
  OI2_CHECK_ARG(groups < 1 << 23, "%d tokens of %d heads are too many for one call", n_tokens, q->heads + k->heads);
  const oi2_heads ko{k_out, k->heads, (int64_t)k->heads * r->head_dim, r->head_dim};
  const int d = r->head_dim;
  OI2_CHECK_ARG(!clashes(true, q_out, q->heads, q, n_tokens, d) && !clashes(true, k_out, k->heads, k, n_tokens, d) &&
                    !clashes(false, q_out, q->heads, k, n_tokens, d) && !clashes(false, k_out, k->heads, q, n_tokens, d) &&
                    !clashes(false, q_out, q->heads, &ko, n_tokens, d),
                "an output shares memory with an input, and is not that input, or with the other output");
  const dim3 grid((uint32_t)groups), block(256);
  hipStream_t st = (hipStream_t)stream;
  const bool bf = dtype == OI2_DTYPE_BF16;
  if (wide && bf) hipLaunchKernelGGL((k_rotary<true, true>), grid, block, 0, st, a);
  else if (wide) hipLaunchKernelGGL((k_rotary<false, true>), grid, block, 0, st, a);
  else if (bf) hipLaunchKernelGGL((k_rotary<true, false>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((k_rotary<false, false>), grid, block, 0, st, a);
  OI2_CHECK_LAUNCH();
  return OI2_OK;
}
