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
// their order does not matter), then takes the slice. Bound by memory, each logit once in and once out, where histories are short
// (256 x 100003 fp32 with a mask each, 41 us: 5.0 TB/s); long ones add their latency (61 us with up to 9000 tokens a row).
// ------------------------------------------------------------------------------------------
struct RulesArgs {
  const void* x;
  void* out;
  int64_t x_row, o_row;
  int rows, vocab, slices;  // blocks of a row
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

// Slices: every block of a row reads its history, so long ones are read for larger slices, of 4096 tokens, or 8192 where there are
// blocks enough; else they are the smallest, of 16 bytes a thread (us with slices of 1024 or 2048 / 4096 / 8192: 1 x 51866 fp16, 224
// tokens 4.8 / 4.3 / 5.2; 40 x 51866, 448 tokens 6.1 / 6.4 / 6.9; 8 x 128000 bf16, up to 30000 tokens 17.3 / 11.3 / 12.9; 256 x 100003
// fp32, no history 41 / 42 / 43, up to 9000 tokens 127 / 73 / 61).
constexpr int64_t kFewMarks = 1024, kFewLogits = int64_t{1} << 23;

// 16 bytes at any element's address.
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
  T e[16 / sizeof(T)];
};

// f(place, token) for the list's places b .. e - 1, a thread's every THREADS-th, kBatch of them requested at once (8 take
// registers that cost blocks a CU: 256 x 100003 fp32 with up to 9000 tokens a row 65 us against 61; with 2 or 3 8 x 128000 bf16 with up
// to 30000 12 to 13 against 11.3).
template <int THREADS, class F>
__device__ __forceinline__ void each_token(const int64_t* tokens, int64_t b, int64_t e, F f) {
  constexpr int kBatch = 4;
  for (int64_t i = b + threadIdx.x; i < e; i += kBatch * THREADS) {
    int64_t t[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) t[j] = tokens[min(i + j * THREADS, e - 1)];
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (i + j * THREADS < e) f(i + j * THREADS, t[j]);
  }
}

// What a slice's cell in LDS says of a token: bit 31 that the prompt has it, bits 16 .. 30 how often it was generated, below 1 + its
// last place in the list of biases. A longer history or list takes two cells, half a slice at a time.
constexpr int64_t kMostMet = 0x7FFF, kMostPlaces = 0xFFFF;

// A slice is V times 16 bytes a thread, which are on their way while the history is counted.
template <class T, int THREADS, int V>
__global__ void __launch_bounds__(THREADS) logits_rules_kernel(RulesArgs a) {
#pragma clang fp contract(off)
  constexpr int kEach = 16 / sizeof(T), kSlice = V * THREADS * kEach;
  extern __shared__ __align__(16) uint32_t cells[];  // [kSlice] where there is a history or a list
  const int row = blockIdx.x / a.slices, from = static_cast<int>(blockIdx.x % a.slices) * kSlice, tid = threadIdx.x;
  const int here = min(kSlice, a.vocab - from);
  const T* x = static_cast<const T*>(a.x) + row * a.x_row + from;
  T* out = static_cast<T*>(a.out) + row * a.o_row + from;
  Loose<T> v[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = kEach * (tid + j * THREADS);
    if (i + kEach <= here) v[j] = *reinterpret_cast<const Loose<T>*>(x + i);
  }
  float repetition = 1.f, presence = 0.f, frequency = 0.f;
  int64_t b = 0, e = 0, made = 0, first = 0, last = 0;
  if (a.tokens) {
    b = within(a.cu[row], 0, a.n_tokens);
    e = within(a.cu[row + 1], b, a.n_tokens);
    made = b + (a.prompt ? within(a.prompt[row], 0, e - b) : 0);
    if (a.repetition) repetition = a.repetition[row];
    if (a.presence) presence = a.presence[row];
    if (a.frequency) frequency = a.frequency[row];
  }
  if (a.bias_ids) {
    first = within(a.cu_bias[row], 0, a.n_bias);
    last = within(a.cu_bias[row + 1], first, a.n_bias);
  }
  const uint32_t* mask = nullptr;
  if (a.masks) {
    const int64_t set = a.mask_of ? a.mask_of[row] : a.n_sets == 1 ? 0 : row;
    if (set >= 0 && set < a.n_sets) mask = a.masks + set * a.mask_row;
  }
  const bool marks = e > b || last > first, split = e - b > kMostMet || last - first > kMostPlaces;
  int64_t listed = first + tid < last ? a.bias_ids[first + tid] : -1;  // on its way too
  // The cells of tokens from .. + [begin, begin + count).
  const auto mark = [&](int begin, int count) {
    for (int i = 4 * tid; i < kSlice; i += 4 * THREADS) *reinterpret_cast<uint4*>(cells + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    each_token<THREADS>(a.tokens, b, e, [&](int64_t i, int64_t token) {
      const int64_t t = token - from - begin;
      if (t < 0 || t >= count) return;
      if (i < made) atomicOr(&cells[t], 0x80000000u);
      else atomicAdd(&cells[t], split ? 1u : 0x10000u);
    });
    if (last > first) {
      __syncthreads();  // the upper bits stay as they are now
      const auto put = [&](int64_t i, int64_t token) {
        const int64_t t = token - from - begin;
        if (t < 0 || t >= count) return;
        const uint32_t place = static_cast<uint32_t>(i - first) + 1;
        if (split) atomicMax(&cells[kSlice / 2 + t], place);
        else atomicMax(&cells[t], (cells[t] & 0xFFFF0000u) | place);
      };
      put(first + tid, listed);
      each_token<THREADS>(a.bias_ids, first + THREADS, last, put);
    }
    __syncthreads();
  };
  const auto rule = [&](T value, uint32_t met, uint32_t count, uint32_t place) {
    float y = static_cast<float>(value);
    if (met) {
      y = y > 0.f ? y / repetition : y * repetition;
      if (count) y = y - frequency * static_cast<float>(count) - presence;
    }
    if (place) y = y + a.bias[first + place - 1];
    return y;
  };
  // (slices begin at multiples of 32 tokens: the bits of a thread's tokens are in one word)
  const auto bits = [&](int i) { return mask ? mask[(from + i) >> 5] >> ((from + i) & 31) : ~0u; };
  if (!split) {
    if (marks) mark(0, here);
    const auto one = [&](T value, int i) {
      const uint32_t cell = marks ? cells[i] : 0;
      return rule(value, cell >> 16, (cell >> 16) & 0x7FFF, cell & 0xFFFF);
    };
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = kEach * (tid + j * THREADS);
      if (i >= here) break;
      const uint32_t may = bits(i);
      if (i + kEach <= here) {
#pragma unroll
        for (int k = 0; k < kEach; ++k) v[j].e[k] = static_cast<T>((may >> k) & 1 ? one(v[j].e[k], i + k) : -INFINITY);
        *reinterpret_cast<Loose<T>*>(out + i) = v[j];
      } else {
        for (int k = 0; i + k < here; ++k) out[i + k] = static_cast<T>((may >> k) & 1 ? one(x[i + k], i + k) : -INFINITY);
      }
    }
    return;
  }
  for (int begin = 0; begin < here; begin += kSlice / 2) {
    const int count = min(kSlice / 2, here - begin);
    if (begin) __syncthreads();  // the half before is done with the cells
    mark(begin, count);
    for (int t = tid; t < count; t += THREADS) {
      const uint32_t cell = cells[t];
      const float y = rule(x[begin + t], cell, cell & 0x7FFFFFFF, cells[kSlice / 2 + t]);
      out[begin + t] = static_cast<T>(bits(begin + t) & 1 ? y : -INFINITY);
    }
  }
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
  RulesArgs a{x, out, x_row, o_row, rows, vocab, 0, tokens, cu, prompt, repetition, presence, frequency,
              bias_ids, bias, cu_bias, n_tokens, n_bias, reinterpret_cast<const uint32_t*>(masks), mask_of, mask_row, n_sets};
  int rc = FW_OK;
  const auto launch = [&](auto kernel, int threads, int slice) {
    a.slices = (vocab + slice - 1) / slice;
    const int64_t blocks = static_cast<int64_t>(rows) * a.slices;
    if (!grid_ok(blocks, threads)) rc = fw_fail(FW_EINVAL, "%s: too many rows", what);
    else hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(threads), tokens || bias_ids ? 4 * slice : 0, stream, a);
  };
  const int64_t each = rows ? (n_tokens + n_bias) / rows : 0, some = static_cast<int64_t>(rows) * vocab;
  const int form = each < kFewMarks ? 0 : some < kFewLogits ? 1 : 2;
  const auto by_size = [&](auto t) {
    typedef decltype(t) T;
    constexpr int kEach = 16 / sizeof(T), kMost = sizeof(T) == 2 ? 2 : 4;
    if (form == 0) launch(logits_rules_kernel<T, 256, 1>, 256, 256 * kEach);
    else if (form == 1) launch(logits_rules_kernel<T, 512, kMost / 2>, 512, 512 * kEach * (kMost / 2));
    else launch(logits_rules_kernel<T, 512, kMost>, 512, 512 * kEach * kMost);
  };
  if (dtype == FW_F16) by_size(_Float16());
  else if (dtype == FW_BF16) by_size(bf16());
  else by_size(0.f);
  if (rc) return rc;
  return fw_check_launch(what);
}
