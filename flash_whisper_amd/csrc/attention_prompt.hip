// Attention over whole prompts for gfx950: sequences of different lengths packed one after another, query
// heads grouped over key/value heads, causal from the end of the keys or not.
#include "fw_common.h"

namespace fw {
namespace {

struct PromptArgs {
  const void *q, *k, *v;
  void* out;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;
  const int64_t *cu_q, *cu_k;
  int64_t q_rows, k_rows;
  int n_seq, heads, kv_heads;
  float scale;
};

// One wave a query and head: a key at a time, D / 64 dims a lane.
template <class T, int D, bool CAUSAL>
__global__ void __launch_bounds__(256) prompt_attention_kernel(PromptArgs a) {
  constexpr int kPer = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6), row = unit / a.heads;
  const int head = static_cast<int>(unit % a.heads), kvh = head / (a.heads / a.kv_heads);
  if (row >= a.q_rows) return;
  int seq = -1;
  for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
    const uint64_t at = __builtin_amdgcn_ballot_w64(s0 + lane < a.n_seq && a.cu_q[min(s0 + lane, a.n_seq)] <= row);
    seq += __popcll(at);
    if (at != ~uint64_t{0}) break;
  }
  if (seq < 0) return;
  const int64_t q0 = max(a.cu_q[seq], int64_t{0}), q1 = min(a.cu_q[seq + 1], a.q_rows);
  if (row >= q1) return;
  const int64_t k0 = min(max(a.cu_k[seq], int64_t{0}), a.k_rows), k1 = min(max(a.cu_k[seq + 1], k0), a.k_rows);
  const int64_t keys = CAUSAL ? min(max(row - q0 + 1 + (k1 - k0) - (q1 - q0), int64_t{0}), k1 - k0) : k1 - k0;
  float q[kPer], acc[kPer] = {}, m = -INFINITY, l = 0.f;
  const T* qp = static_cast<const T*>(a.q) + row * a.q_row + head * a.q_head;
  for (int i = 0; i < kPer; ++i) q[i] = static_cast<float>(qp[lane + 64 * i]) * a.scale;
  for (int64_t t = k0; t < k0 + keys; ++t) {
    const T* kp = static_cast<const T*>(a.k) + t * a.k_row + kvh * a.k_head;
    const T* vp = static_cast<const T*>(a.v) + t * a.v_row + kvh * a.v_head;
    float s = 0.f;
    for (int i = 0; i < kPer; ++i) s += q[i] * static_cast<float>(kp[lane + 64 * i]);
    s = group_sum<64>(s);
    const float m_new = fmaxf(m, s), corr = __expf(m - m_new), p = __expf(s - m_new);
    l = l * corr + p;
    for (int i = 0; i < kPer; ++i) acc[i] = acc[i] * corr + p * static_cast<float>(vp[lane + 64 * i]);
    m = m_new;
  }
  T* op = static_cast<T*>(a.out) + row * a.o_row + head * a.o_head;
  for (int i = 0; i < kPer; ++i) op[lane + 64 * i] = static_cast<T>(keys > 0 ? acc[i] / l : 0.f);
}

bool rows_ok(const void* p, int64_t row, int64_t head) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && row % 8 == 0 && head % 8 == 0;
}

}  // namespace
}  // namespace fw

using namespace fw;

extern "C" int fw_prompt_attention(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                                   const void* v, int64_t v_row, int64_t v_head, void* out, int64_t o_row, int64_t o_head,
                                   const int64_t* cu_q, const int64_t* cu_k, int n_seq, int64_t q_rows, int64_t k_rows,
                                   int heads, int kv_heads, int head_dim, int dtype, float scale, int causal,
                                   hipStream_t stream) {
  if (n_seq <= 0 || q_rows < 0 || k_rows < 0) return fw_fail(FW_EINVAL, "prompt_attention: n_seq must be positive, rows not negative");
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads) return fw_fail(FW_EINVAL, "prompt_attention: heads must be a multiple of kv_heads");
  if (head_dim != 64 && head_dim != 128) return fw_fail(FW_EINVAL, "prompt_attention: head_dim must be 64 or 128");
  if (dtype != FW_F16 && dtype != FW_BF16) return fw_fail(FW_EINVAL, "prompt_attention: dtype must be FW_F16 or FW_BF16");
  if (!cu_q || !cu_k || (q_rows > 0 && (!q || !out)) || (k_rows > 0 && (!k || !v)))
    return fw_fail(FW_EINVAL, "prompt_attention: null pointer");
  if ((q_rows > 0 && (!rows_ok(q, q_row, q_head) || !rows_ok(out, o_row, o_head))) ||
      (k_rows > 0 && (!rows_ok(k, k_row, k_head) || !rows_ok(v, v_row, v_head))))
    return fw_fail(FW_EINVAL, "prompt_attention: q, k, v and out must be 16-byte aligned with strides in multiples of 8");
  if (q_rows == 0) return FW_OK;
  const PromptArgs a{q, k, v, out, q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head, cu_q, cu_k, q_rows, k_rows, n_seq, heads, kv_heads, scale};
  const int64_t blocks = (q_rows * heads + 3) / 4;
  if (blocks > 0x7FFFFFFF) return fw_fail(FW_EINVAL, "prompt_attention: too many rows");
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, a);
  };
  const auto by_mask = [&](auto full, auto masked) { causal ? launch(masked) : launch(full); };
  if (dtype == FW_F16 && head_dim == 64) by_mask(prompt_attention_kernel<_Float16, 64, false>, prompt_attention_kernel<_Float16, 64, true>);
  else if (dtype == FW_F16) by_mask(prompt_attention_kernel<_Float16, 128, false>, prompt_attention_kernel<_Float16, 128, true>);
  else if (head_dim == 64) by_mask(prompt_attention_kernel<__bf16, 64, false>, prompt_attention_kernel<__bf16, 64, true>);
  else by_mask(prompt_attention_kernel<__bf16, 128, false>, prompt_attention_kernel<__bf16, 128, true>);
  return fw_check_launch("prompt_attention");
}
