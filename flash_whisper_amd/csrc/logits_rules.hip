// Rules on the logits of a batch for gfx950: penalties for the tokens of a row's history, biases, the mask of a grammar.
#include "packed_rows.h"

namespace fw {
namespace {

typedef __bf16 bf16;

// ------------------------------------------------------------------------------------------
// Of row r and token i, in fp32 and in this order, rounded once at the end:
//   x <- x / repetition[r] if x > 0, else x repetition[r], for a token of the row's history
//   x <- x - frequency[r] c - presence[r] for one that comes c > 0 times behind the history's first prompt[r] tokens
//   x <- x + b, b the bias of the token's last place in the row's list
//   x <- -infinity where the token's bit in the row's mask is 0
// A block has a slice of a row. It counts the history's and the list's tokens that fall into the slice in LDS (whole numbers, so
// their order does not matter), then takes the slice 16 bytes a thread. Bound by memory: each logit once in and once out.
// ------------------------------------------------------------------------------------------
struct RulesArgs {
  const void* x;
  void* out;
  int64_t x_row, o_row;
  int rows, vocab, slice, slices;
  const int64_t *tokens, *cu, *prompt;
  const float *repetition, *presence, *frequency;
  const int64_t* bias_ids;
  const float* bias;
  const int64_t* cu_bias;
  int64_t n_tokens, n_bias;
  const uint32_t* masks;
  const int64_t* mask_of;
  int64_t mask_row;
  int n_sets;
};

constexpr int kThreads = 256;
constexpr uint32_t kMet = 0x80000000u;  // a token of the prompt; below: how often it was generated

// 16 bytes at any element's address.
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
  T e[16 / sizeof(T)];
};

template <class T>
__global__ void __launch_bounds__(kThreads) logits_rules_kernel(RulesArgs a) {
#pragma clang fp contract(off)
  constexpr int kEach = 16 / sizeof(T);
  extern __shared__ __align__(16) uint32_t lds[];
  const int row = blockIdx.x / a.slices, begin = blockIdx.x % a.slices * a.slice, tid = threadIdx.x;
  const int count = min(a.slice, a.vocab - begin);
  uint32_t* met = lds;                                // [slice] if there is a history
  uint32_t* place = lds + (a.tokens ? a.slice : 0);   // [slice] if there are biases: 1 + the last place in the list
  const int words = (a.tokens ? a.slice : 0) + (a.bias_ids ? a.slice : 0);
  for (int i = 4 * tid; i < words; i += 4 * kThreads) *reinterpret_cast<uint4*>(lds + i) = make_uint4(0, 0, 0, 0);
  if (words) __syncthreads();
  float repetition = 1.f, presence = 0.f, frequency = 0.f;
  if (a.tokens) {
    const int64_t b = within(a.cu[row], 0, a.n_tokens), e = within(a.cu[row + 1], b, a.n_tokens);
    const int64_t made = b + (a.prompt ? within(a.prompt[row], 0, e - b) : 0);
    if (a.repetition) repetition = a.repetition[row];
    if (a.presence) presence = a.presence[row];
    if (a.frequency) frequency = a.frequency[row];
    for (int64_t i = b + tid; i < e; i += kThreads) {
      const int64_t t = a.tokens[i] - begin;
      if (t < 0 || t >= count) continue;
      if (i < made) atomicOr(&met[t], kMet);
      else atomicAdd(&met[t], 1u);
    }
  }
  int64_t first = 0;
  if (a.bias_ids) {
    first = within(a.cu_bias[row], 0, a.n_bias);
    const int64_t e = within(a.cu_bias[row + 1], first, a.n_bias);
    for (int64_t i = first + tid; i < e; i += kThreads) {
      const int64_t t = a.bias_ids[i] - begin;
      if (t >= 0 && t < count) atomicMax(&place[t], static_cast<uint32_t>(i - first) + 1);
    }
  }
  if (words) __syncthreads();
  const uint32_t* mask = nullptr;
  if (a.masks) {
    const int64_t set = a.mask_of ? a.mask_of[row] : a.n_sets == 1 ? 0 : row;
    if (set >= 0 && set < a.n_sets) mask = a.masks + set * a.mask_row;
  }
  const T* x = static_cast<const T*>(a.x) + row * a.x_row + begin;
  T* out = static_cast<T*>(a.out) + row * a.o_row + begin;
  const auto rule = [&](T value, int i) {
    float y = static_cast<float>(value);
    if (a.tokens) {
      const uint32_t m = met[i], c = m & ~kMet;
      if (m) {
        y = y > 0.f ? y / repetition : y * repetition;
        if (c) y = y - frequency * static_cast<float>(c) - presence;
      }
    }
    if (a.bias_ids && place[i]) y = y + a.bias[first + place[i] - 1];
    return y;
  };
  for (int i = kEach * tid; i < count; i += kEach * kThreads) {
    // (slices begin at multiples of 32 tokens: the bits of a thread's tokens are in one word)
    const uint32_t may = mask ? mask[(begin + i) >> 5] >> ((begin + i) & 31) : ~0u;
    if (i + kEach <= count) {
      Loose<T> v = *reinterpret_cast<const Loose<T>*>(x + i);
#pragma unroll
      for (int e = 0; e < kEach; ++e) v.e[e] = static_cast<T>((may >> e) & 1 ? rule(v.e[e], i + e) : -INFINITY);
      *reinterpret_cast<Loose<T>*>(out + i) = v;
    } else {
      for (int e = 0; i + e < count; ++e) out[i + e] = static_cast<T>((may >> e) & 1 ? rule(x[i + e], i + e) : -INFINITY);
    }
  }
}

// Tokens of a slice: few where there are few rows, so that more CUs have one.
int rules_slice(int rows, int vocab) {
  return static_cast<int64_t>(rows) * vocab < (int64_t{1} << 22) ? 2048 : 4096;
}

}  // namespace
}  // namespace fw

using namespace fw;

extern "C" int fw_logits_rules(const void* x, int64_t x_row, void* out, int64_t o_row, int rows, int vocab, int dtype,
                               const int64_t* tokens, int64_t n_tokens, const int64_t* cu, const int64_t* prompt,
                               const float* repetition, const float* presence, const float* frequency,
                               const int64_t* bias_ids, const float* bias, int64_t n_bias, const int64_t* cu_bias,
                               const int32_t* masks, int64_t mask_row, int n_sets, const int64_t* mask_of,
                               hipStream_t stream) {
  const char* what = "logits_rules";
  if (dtype != FW_F16 && dtype != FW_BF16 && dtype != FW_F32)
    return fw_fail(FW_EINVAL, "%s: dtype must be FW_F16, FW_BF16 or FW_F32", what);
  if (rows < 0 || vocab <= 0 || vocab > 0x7FFF0000) return fw_fail(FW_EINVAL, "%s: rows must not be negative, vocab positive", what);
  if (n_tokens < 0 || n_bias < 0 || n_bias > 0x7FFFFFFF) return fw_fail(FW_EINVAL, "%s: too many or negative tokens or biases", what);
  if (rows > 0 && (!x || !out)) return fw_fail(FW_EINVAL, "%s: null pointer", what);
  if (!cu != !tokens || ((prompt || repetition || presence || frequency) && !tokens))
    return fw_fail(FW_EINVAL, "%s: penalties need tokens and their starts", what);
  if (!bias_ids != !bias || !bias_ids != !cu_bias)
    return fw_fail(FW_EINVAL, "%s: bias_ids, bias and cu_bias must be given together", what);
  if ((mask_of && !masks) || (masks && (n_sets <= 0 || mask_row < (static_cast<int64_t>(vocab) + 31) / 32 ||
                                        (!mask_of && n_sets != 1 && n_sets < rows))))
    return fw_fail(FW_EINVAL, "%s: masks must hold vocab bits for each set, and a set for each row or one for all", what);
  if (rows == 0) return FW_OK;
  RulesArgs a{x, out, x_row, o_row, rows, vocab, rules_slice(rows, vocab), 0, tokens, cu, prompt, repetition, presence, frequency,
              bias_ids, bias, cu_bias, n_tokens, n_bias, reinterpret_cast<const uint32_t*>(masks), mask_of, mask_row, n_sets};
  a.slices = (vocab + a.slice - 1) / a.slice;
  const int64_t blocks = static_cast<int64_t>(rows) * a.slices;
  if (!grid_ok(blocks, kThreads)) return fw_fail(FW_EINVAL, "%s: too many rows", what);
  const int lds = 4 * a.slice * ((tokens != nullptr) + (bias_ids != nullptr));
  const auto kernel = dtype == FW_F16 ? logits_rules_kernel<_Float16> : dtype == FW_BF16 ? logits_rules_kernel<bf16> : logits_rules_kernel<float>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), lds, stream, a);
  return fw_check_launch(what);
}
