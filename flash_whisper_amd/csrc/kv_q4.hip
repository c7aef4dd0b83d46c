// Key/value cache held in 4 bits for gfx950: rows written into it, read back, and the single-token
// attention over it. Layout (L = max_len, a multiple of 32; D = 64 or 128; 32 dims of a row, a group,
// share a step and a low value):
//   k_codes [seq][head][L][D / 2]          row-major: lane = key of the score products
//   k_meta  [seq][head][L][D / 32] {step, low}
//   v_codes [seq][head][L / 8][D / 4][16]  8 rows x 4 dims in 16 bytes, row t's 4 dims at byte 2 (t % 8):
//                                          one 16-byte load holds a lane's 8 keys of the P V products
//   v_meta  [seq][head][L / 8][D / 32] {step of 8 rows, low of 8 rows}
// A code c stands for fp16(low + step c), one rounding; 5 bits a value with step and low.
#include "fw_common.h"

namespace fw {
namespace {

typedef unsigned short u16;

struct Q4Cache {
  uint8_t* k_codes;
  _Float16* k_meta;
  uint8_t* v_codes;
  _Float16* v_meta;
  int n_seq, heads, max_len;
};

// Rows k, v [tokens, heads, D] with their element strides.
struct Q4Rows {
  const void *k, *v;
  int64_t k_row, k_head, v_row, v_head;
};

template <class T>
struct Vec8 {
  typedef T type __attribute__((ext_vector_type(8)));
};

// ------------------------------------------------------------------------------------------
// Which packed rows a wave works on. The rows of sequence s go to cache rows pos[s] .. and a wave takes one
// aligned block of 8 cache rows, so that the 16-byte units of V are written whole. Sequence s owns the
// wave slots from cu[s] / 8 + 2 s on: its rows touch at most floor((len + 14) / 8) blocks, and the next
// sequence's slots begin at least floor(len / 8) + 2 later.
// ------------------------------------------------------------------------------------------
struct Q4Slot {
  int seq;        // -1: nothing to do
  int64_t first;  // packed row of cache row `row` (may lie before the sequence's own rows)
  int64_t begin, end;  // the sequence's packed rows
  int64_t row;    // first cache row of the block, a multiple of 8 (may be negative or past the cache)
};

__device__ __forceinline__ Q4Slot q4_slot(const int64_t* cu, const int64_t* pos, int n_seq, int64_t rows, int64_t slot) {
  const int lane = threadIdx.x & 63;
  int seq = -1;
  for (int s0 = 0; s0 < n_seq; s0 += 64) {  // the last sequence whose slots begin at or before this one
    const int s = s0 + lane;
    const int64_t c = s < n_seq ? min(max(cu[s], int64_t{0}), rows) : rows;
    const uint64_t at = __builtin_amdgcn_ballot_w64(s < n_seq && c / 8 + 2 * static_cast<int64_t>(s) <= slot);
    seq += __popcll(at);
    if (at != ~uint64_t{0}) break;
  }
  Q4Slot r{seq, 0, 0, 0, 0};
  if (seq < 0) return r;
  r.begin = min(max(cu[seq], int64_t{0}), rows);
  r.end = min(max(cu[seq + 1], r.begin), rows);
  const int64_t p = pos[seq], block = slot - (r.begin / 8 + 2 * static_cast<int64_t>(seq));
  r.row = (p & ~int64_t{7}) + 8 * block;
  r.first = r.begin + (r.row - p);
  if (r.first >= r.end) r.seq = -1;
  return r;
}

// A group's step and low from its smallest and largest value: the step rounded towards zero, so that
// low + 15 step stays within the group's values and no finite value reads back as an infinity. A group
// holding a NaN or an infinity gets a NaN step and reads back as NaN.
__device__ __forceinline__ void q4_meta(float lo, float hi, bool finite, _Float16& step, _Float16& low) {
  const auto rtz = __builtin_amdgcn_cvt_pkrtz((hi - lo) * (1.0f / 15.0f), 0.f);
  step = finite ? static_cast<_Float16>(rtz[0]) : static_cast<_Float16>(__builtin_nanf(""));
  low = f2h(lo);
}

// The nearest code of x, ties to the even one: the rounded quotient by the reciprocal is at most one off, and
// the remainder, which fma gives with one rounding, says where.
__device__ __forceinline__ uint32_t q4_code(float x, float low, float step, float inverse) {
  const float d = x - low;
  float c = rintf(d * inverse);
  const float rest = fmaf(-c, step, d), half = 0.5f * step;
  const bool odd = (static_cast<int>(c) & 1) != 0;
  if (rest > half || (rest == half && odd)) c += 1.f;
  else if (rest < -half || (rest == -half && odd)) c -= 1.f;
  return static_cast<uint32_t>(fminf(fmaxf(c, 0.f), 15.f));
}

// 8 values of a lane to 8 codes in a dword, element e in bits 4 e; the 4 lanes of a group agree on its meta.
template <class T>
__device__ __forceinline__ uint32_t q4_pack8(const typename Vec8<T>::type& x, _Float16& step, _Float16& low) {
  float f[8], lo = INFINITY, hi = -INFINITY;
  bool finite = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f[e] = static_cast<float>(x[e]);
    finite = finite && __builtin_fabsf(f[e]) < INFINITY;
    lo = fminf(lo, f[e]);
    hi = fmaxf(hi, f[e]);
  }
  lo = -xor_max<1>(xor_max<2>(-lo));
  hi = xor_max<1>(xor_max<2>(hi));
  finite = xor_max<1>(xor_max<2>(finite ? 0.f : 1.f)) == 0.f;
  q4_meta(lo, hi, finite, step, low);
  const float s = h2f(step), l = h2f(low), inverse = s > 0.f ? 1.0f / s : 0.f;
  uint32_t codes = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) codes |= (s > 0.f ? q4_code(f[e], l, s, inverse) : 0u) << (4 * e);
  return codes;
}

// ------------------------------------------------------------------------------------------
// Append: a wave = 8 cache rows x 64 dims of a head (lane = row lane / 8, dims 8 (lane % 8)), K and V. Bound
// by memory: 2 x 2 bytes a value pair in, 2 x 0.625 out. K leaves as one dword a lane (whole rows); V's 2-byte
// pieces of 8 rows meet in LDS and leave as one dword a lane where all 8 rows are written, and piece by
// piece at a sequence's ends, where the other rows of the unit stay as they are.
// ------------------------------------------------------------------------------------------
template <class T, int D>
__global__ void __launch_bounds__(256) kv_q4_append_kernel(Q4Rows in, const int64_t* __restrict__ cu,
                                                           const int64_t* __restrict__ pos, int64_t rows, int64_t slots,
                                                           Q4Cache c) {
  __shared__ __align__(16) u16 pieces[4][16][8];
  constexpr int kHalves = D / 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  const int part = static_cast<int>(unit % (c.heads * kHalves)), head = part / kHalves, d0 = part % kHalves * 64;
  const int64_t slot = unit / (c.heads * kHalves);
  if (slot >= slots) return;  // no block barrier below
  const Q4Slot w = q4_slot(cu, pos, c.n_seq, rows, slot);
  if (w.seq < 0) return;
  const int r = lane >> 3, d = d0 + 8 * (lane & 7);
  const int64_t token = w.first + r, row = w.row + r;
  const bool live = token >= w.begin && token < w.end && row >= 0 && row < c.max_len;
  const bool whole = __builtin_amdgcn_ballot_w64(live) == ~uint64_t{0};
  typename Vec8<T>::type kx = {}, vx = {};
  if (live) {
    kx = *reinterpret_cast<const typename Vec8<T>::type*>(static_cast<const T*>(in.k) + token * in.k_row + head * in.k_head + d);
    vx = *reinterpret_cast<const typename Vec8<T>::type*>(static_cast<const T*>(in.v) + token * in.v_row + head * in.v_head + d);
  }
  _Float16 ks, kl, vs, vl;
  const uint32_t kc = q4_pack8<T>(kx, ks, kl), vc = q4_pack8<T>(vx, vs, vl);
  const int64_t hr = (static_cast<int64_t>(w.seq) * c.heads + head) * c.max_len;  // the head's first row
  if (live) {
    const int64_t at = hr + row;
    *reinterpret_cast<uint32_t*>(c.k_codes + at * (D / 2) + d / 2) = kc;
    if ((lane & 3) == 0) {
      *reinterpret_cast<h2v*>(c.k_meta + (at * (D / 32) + d / 32) * 2) = h2v{ks, kl};
      _Float16* vm = c.v_meta + (((hr + w.row) / 8 * (D / 32) + d / 32) * 2) * 8;
      vm[r] = vs;
      vm[8 + r] = vl;
    }
  }
  uint8_t* vu = c.v_codes + (hr + w.row) / 8 * (D / 4) * 16 + static_cast<int64_t>(d0 / 4) * 16;
  if (whole) {
    u16(*p)[8] = pieces[wave];
    p[2 * (lane & 7)][r] = static_cast<u16>(vc);
    p[2 * (lane & 7) + 1][r] = static_cast<u16>(vc >> 16);
    __builtin_amdgcn_wave_barrier();  // one wave's own LDS accesses stay in order
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    reinterpret_cast<uint32_t*>(vu)[lane] = reinterpret_cast<const uint32_t*>(&p[0][0])[lane];
  } else if (live) {
    *reinterpret_cast<u16*>(vu + (2 * (lane & 7)) * 16 + 2 * r) = static_cast<u16>(vc);
    *reinterpret_cast<u16*>(vu + (2 * (lane & 7) + 1) * 16 + 2 * r) = static_cast<u16>(vc >> 16);
  }
}

// ------------------------------------------------------------------------------------------
// Read: the rows that an append of the same cu and pos wrote, as the values that they stand for. Waves and
// lanes as in the append; rows outside the cache read as zeros.
// ------------------------------------------------------------------------------------------
template <class T>
__device__ __forceinline__ typename Vec8<T>::type q4_values8(uint32_t codes, _Float16 step, _Float16 low) {
  typename Vec8<T>::type x;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const _Float16 c = static_cast<_Float16>(static_cast<float>((codes >> (4 * e)) & 15u));
    x[e] = static_cast<T>(h2f(__builtin_fmaf16(c, step, low)));
  }
  return x;
}

template <class T, int D>
__global__ void __launch_bounds__(256) kv_q4_read_kernel(Q4Rows out, const int64_t* __restrict__ cu,
                                                         const int64_t* __restrict__ pos, int64_t rows, int64_t slots,
                                                         Q4Cache c) {
  constexpr int kHalves = D / 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  const int part = static_cast<int>(unit % (c.heads * kHalves)), head = part / kHalves, d0 = part % kHalves * 64;
  const int64_t slot = unit / (c.heads * kHalves);
  if (slot >= slots) return;
  const Q4Slot w = q4_slot(cu, pos, c.n_seq, rows, slot);
  if (w.seq < 0) return;
  const int r = lane >> 3, d = d0 + 8 * (lane & 7);
  const int64_t token = w.first + r, row = w.row + r;
  if (token < w.begin || token >= w.end) return;
  const int64_t hr = (static_cast<int64_t>(w.seq) * c.heads + head) * c.max_len;
  typename Vec8<T>::type kx = {}, vx = {};
  if (row >= 0 && row < c.max_len) {
    const int64_t at = hr + row, block = (hr + w.row) / 8;
    const h2v km = *reinterpret_cast<const h2v*>(c.k_meta + (at * (D / 32) + d / 32) * 2);
    kx = q4_values8<T>(*reinterpret_cast<const uint32_t*>(c.k_codes + at * (D / 2) + d / 2), km[0], km[1]);
    const uint8_t* vu = c.v_codes + (block * (D / 4) + d / 4) * 16 + 2 * r;
    const uint32_t vc = *reinterpret_cast<const u16*>(vu) | static_cast<uint32_t>(*reinterpret_cast<const u16*>(vu + 16)) << 16;
    const _Float16* vm = c.v_meta + (block * (D / 32) + d / 32) * 16;
    vx = q4_values8<T>(vc, vm[r], vm[8 + r]);
  }
  T* ko = static_cast<T*>(const_cast<void*>(out.k)) + token * out.k_row + head * out.k_head + d;
  T* vo = static_cast<T*>(const_cast<void*>(out.v)) + token * out.v_row + head * out.v_head + d;
  *reinterpret_cast<typename Vec8<T>::type*>(ko) = kx;
  *reinterpret_cast<typename Vec8<T>::type*>(vo) = vx;
}

// ------------------------------------------------------------------------------------------
// Single-token attention: block = (sequence, query head), 4 waves; a wave takes a key at a time, lanes hold
// D / 64 dims each. The fresh row of the head is written first by the block itself.
// ------------------------------------------------------------------------------------------
struct Q4Attn {
  const void* q;
  void* out;
  int64_t q_row, q_head, o_row, o_head;
  Q4Rows fresh;  // k_new, v_new [seq, kv head, D], or null
  const int64_t* lens;
  Q4Cache c;
  int heads;  // query heads
  float scale;
};

// Row `row` of a head from its fresh values: waves 0 and 1 write K and V, lane = dims {lane, lane + 64}.
template <class T, int D>
__device__ __forceinline__ void q4_write_row(const Q4Attn& a, int seq, int kvh, int row, int wave, int lane) {
  if (wave > 1) return;
  const Q4Cache& c = a.c;
  const int64_t hr = (static_cast<int64_t>(seq) * c.heads + kvh) * c.max_len;
  const T* src = wave == 0 ? static_cast<const T*>(a.fresh.k) + seq * a.fresh.k_row + kvh * a.fresh.k_head
                           : static_cast<const T*>(a.fresh.v) + seq * a.fresh.v_row + kvh * a.fresh.v_head;
#pragma unroll
  for (int h = 0; h < D / 64; ++h) {
    const int d = 64 * h + 8 * (lane & 7);  // every 8 lanes do the same; the first 8 store
    _Float16 step, low;
    const uint32_t codes = q4_pack8<T>(*reinterpret_cast<const typename Vec8<T>::type*>(src + d), step, low);
    if (lane >= 8) continue;
    if (wave == 0) {
      *reinterpret_cast<uint32_t*>(c.k_codes + (hr + row) * (D / 2) + d / 2) = codes;
      if ((lane & 3) == 0) *reinterpret_cast<h2v*>(c.k_meta + ((hr + row) * (D / 32) + d / 32) * 2) = h2v{step, low};
    } else {
      const int64_t block = hr / 8 + row / 8;
      uint8_t* vu = c.v_codes + (block * (D / 4) + d / 4) * 16 + 2 * (row & 7);
      *reinterpret_cast<u16*>(vu) = static_cast<u16>(codes);
      *reinterpret_cast<u16*>(vu + 16) = static_cast<u16>(codes >> 16);
      if ((lane & 3) == 0) {
        _Float16* vm = c.v_meta + (block * (D / 32) + d / 32) * 16 + (row & 7);
        vm[0] = step;
        vm[8] = low;
      }
    }
  }
}

// Cached keys of a sequence, and the row that a fresh token goes to (-1: none). A negative length is an idle
// sequence; a full cache has its last row overwritten, as the position of the batch-1 decoder stays at its
// last one.
__device__ __forceinline__ int q4_keys(const Q4Attn& a, int seq, int& fresh_row) {
  const int64_t len = a.lens[seq];
  fresh_row = -1;
  if (len < 0) return 0;
  if (!a.fresh.k) return static_cast<int>(min(len, static_cast<int64_t>(a.c.max_len)));
  fresh_row = static_cast<int>(min(len, static_cast<int64_t>(a.c.max_len - 1)));
  return fresh_row + 1;
}

template <class T, int D>
__global__ void __launch_bounds__(256) decode_attention_q4_kernel(Q4Attn a) {
  constexpr int kPer = D / 64;
  __shared__ float sm[4], sl[4], sacc[4][D];
  const int seq = blockIdx.y, head = blockIdx.x, kvh = head / (a.heads / a.c.heads);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int fresh;
  const int keys = q4_keys(a, seq, fresh);
  if (fresh >= 0) {
    q4_write_row<T, D>(a, seq, kvh, fresh, wave, lane);
    __syncthreads();
  }
  const int64_t hr = (static_cast<int64_t>(seq) * a.c.heads + kvh) * a.c.max_len;
  float q[kPer], acc[kPer] = {}, m = -INFINITY, l = 0.f;
  const T* qp = static_cast<const T*>(a.q) + seq * a.q_row + head * a.q_head;
  for (int i = 0; i < kPer; ++i) q[i] = static_cast<float>(qp[lane + 64 * i]) * a.scale;
  for (int t = wave; t < keys; t += 4) {
    float s = 0.f, v[kPer];
    for (int i = 0; i < kPer; ++i) {
      const int d = lane + 64 * i, sh = 4 * (d & 1);
      const _Float16* km = a.c.k_meta + ((hr + t) * (D / 32) + d / 32) * 2;
      const float kc = static_cast<float>((a.c.k_codes[(hr + t) * (D / 2) + d / 2] >> sh) & 15);
      s += q[i] * h2f(__builtin_fmaf16(static_cast<_Float16>(kc), km[0], km[1]));
      const int64_t block = hr / 8 + t / 8;
      const _Float16* vm = a.c.v_meta + (block * (D / 32) + d / 32) * 16 + (t & 7);
      const float vc = static_cast<float>((a.c.v_codes[(block * (D / 4) + d / 4) * 16 + 2 * (t & 7) + (d & 3) / 2] >> sh) & 15);
      v[i] = h2f(__builtin_fmaf16(static_cast<_Float16>(vc), vm[0], vm[8]));
    }
    s = group_sum<64>(s);
    const float m_new = fmaxf(m, s), corr = __expf(m - m_new), p = __expf(s - m_new);
    l = l * corr + p;
    for (int i = 0; i < kPer; ++i) acc[i] = acc[i] * corr + p * v[i];
    m = m_new;
  }
  if (lane == 0) {
    sm[wave] = m;
    sl[wave] = l;
  }
  for (int i = 0; i < kPer; ++i) sacc[wave][lane + 64 * i] = acc[i];
  __syncthreads();
  if (threadIdx.x >= D) return;
  float top = -INFINITY, num = 0.f, den = 0.f;
  for (int w = 0; w < 4; ++w) top = fmaxf(top, sm[w]);
  for (int w = 0; w < 4; ++w) {
    if (sl[w] == 0.f) continue;
    const float e = __expf(sm[w] - top);
    num += e * sacc[w][threadIdx.x];
    den += e * sl[w];
  }
  static_cast<T*>(a.out)[seq * a.o_row + head * a.o_head + threadIdx.x] = static_cast<T>(den > 0.f ? num / den : 0.f);
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// What every entry point asks of a cache; FW_OK or FW_EINVAL.
int check_cache(const char* what, const Q4Cache& c, int dim) {
  if (!c.k_codes || !c.k_meta || !c.v_codes || !c.v_meta) return fw_fail(FW_EINVAL, "%s: null cache pointer", what);
  if (c.n_seq <= 0 || c.heads <= 0) return fw_fail(FW_EINVAL, "%s: n_seq and kv_heads must be positive", what);
  if (dim != 64 && dim != 128) return fw_fail(FW_EINVAL, "%s: head_dim must be 64 or 128", what);
  if (c.max_len <= 0 || c.max_len % 32) return fw_fail(FW_EINVAL, "%s: max_len must be a positive multiple of 32", what);
  if (!aligned(c.k_codes, 16) || !aligned(c.k_meta, 16) || !aligned(c.v_codes, 16) || !aligned(c.v_meta, 16))
    return fw_fail(FW_EINVAL, "%s: the cache must be 16-byte aligned", what);
  return FW_OK;
}

// Rows whose 8-element pieces are 16-byte accesses.
bool rows_ok(const void* p, int64_t row, int64_t head) { return aligned(p, 16) && row % 8 == 0 && head % 8 == 0; }

// kernel<T, D> for a dtype and a head size.
#define Q4_LAUNCH(kernel, dtype, dim, grid, block, stream, ...)                                           \
  do {                                                                                                    \
    if ((dtype) == FW_F16 && (dim) == 64) hipLaunchKernelGGL((kernel<_Float16, 64>), grid, block, 0, stream, __VA_ARGS__); \
    else if ((dtype) == FW_F16) hipLaunchKernelGGL((kernel<_Float16, 128>), grid, block, 0, stream, __VA_ARGS__);          \
    else if ((dim) == 64) hipLaunchKernelGGL((kernel<__bf16, 64>), grid, block, 0, stream, __VA_ARGS__);  \
    else hipLaunchKernelGGL((kernel<__bf16, 128>), grid, block, 0, stream, __VA_ARGS__);                  \
  } while (0)

int check_packed(const char* what, const Q4Rows& r, const int64_t* cu, const int64_t* pos, int64_t rows, const Q4Cache& c,
                 int dim, int dtype) {
  if (const int rc = check_cache(what, c, dim)) return rc;
  if (dtype != FW_F16 && dtype != FW_BF16) return fw_fail(FW_EINVAL, "%s: dtype must be FW_F16 or FW_BF16", what);
  if (rows < 0) return fw_fail(FW_EINVAL, "%s: rows must not be negative", what);
  if (!cu || !pos || (rows > 0 && (!r.k || !r.v))) return fw_fail(FW_EINVAL, "%s: null pointer", what);
  if (rows > 0 && (!rows_ok(r.k, r.k_row, r.k_head) || !rows_ok(r.v, r.v_row, r.v_head)))
    return fw_fail(FW_EINVAL, "%s: k and v must be 16-byte aligned with strides in multiples of 8", what);
  // the grid: 4 waves a block, slots x heads x halves waves
  if ((rows / 8 + 2 * static_cast<int64_t>(c.n_seq)) * c.heads * (dim / 64) > int64_t{4} * 0x7FFFFFFF)
    return fw_fail(FW_EINVAL, "%s: too many rows", what);
  return FW_OK;
}

}  // namespace
}  // namespace fw

using namespace fw;

extern "C" int fw_kv_q4_append(const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                               int64_t rows, const int64_t* cu, const int64_t* pos, void* k_codes, void* k_meta,
                               void* v_codes, void* v_meta, int n_seq, int kv_heads, int max_len, int head_dim, int dtype,
                               hipStream_t stream) {
  const Q4Cache c{static_cast<uint8_t*>(k_codes), static_cast<_Float16*>(k_meta), static_cast<uint8_t*>(v_codes),
                  static_cast<_Float16*>(v_meta), n_seq, kv_heads, max_len};
  const Q4Rows r{k, v, k_row, k_head, v_row, v_head};
  if (const int rc = check_packed("kv_q4_append", r, cu, pos, rows, c, head_dim, dtype)) return rc;
  if (rows == 0) return FW_OK;
  const int64_t slots = rows / 8 + 2 * static_cast<int64_t>(n_seq), units = slots * kv_heads * (head_dim / 64);
  Q4_LAUNCH(kv_q4_append_kernel, dtype, head_dim, dim3(static_cast<unsigned>((units + 3) / 4)), dim3(256), stream, r, cu,
            pos, rows, slots, c);
  return fw_check_launch("kv_q4_append");
}

extern "C" int fw_kv_q4_read(const void* k_codes, const void* k_meta, const void* v_codes, const void* v_meta, int n_seq,
                             int kv_heads, int max_len, int head_dim, const int64_t* cu, const int64_t* pos, int64_t rows,
                             void* k, int64_t k_row, int64_t k_head, void* v, int64_t v_row, int64_t v_head, int dtype,
                             hipStream_t stream) {
  const Q4Cache c{static_cast<uint8_t*>(const_cast<void*>(k_codes)), static_cast<_Float16*>(const_cast<void*>(k_meta)),
                  static_cast<uint8_t*>(const_cast<void*>(v_codes)), static_cast<_Float16*>(const_cast<void*>(v_meta)),
                  n_seq, kv_heads, max_len};
  const Q4Rows r{k, v, k_row, k_head, v_row, v_head};
  if (const int rc = check_packed("kv_q4_read", r, cu, pos, rows, c, head_dim, dtype)) return rc;
  if (rows == 0) return FW_OK;
  const int64_t slots = rows / 8 + 2 * static_cast<int64_t>(n_seq), units = slots * kv_heads * (head_dim / 64);
  Q4_LAUNCH(kv_q4_read_kernel, dtype, head_dim, dim3(static_cast<unsigned>((units + 3) / 4)), dim3(256), stream, r, cu,
            pos, rows, slots, c);
  return fw_check_launch("kv_q4_read");
}

extern "C" int64_t fw_decode_attention_q4_ws_floats(int n_seq, int heads, int kv_heads, int max_len, int head_dim) {
  if (n_seq <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || max_len <= 0 || max_len % 32 ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  return 4;
}

extern "C" int fw_decode_attention_q4(const void* q, int64_t q_row, int64_t q_head, void* k_codes, void* k_meta,
                                      void* v_codes, void* v_meta, const int64_t* lens, void* out, int64_t o_row,
                                      int64_t o_head, const void* k_new, int64_t k_row, int64_t k_head, const void* v_new,
                                      int64_t v_row, int64_t v_head, int n_seq, int heads, int kv_heads, int max_len,
                                      int head_dim, int dtype, float scale, float* ws, int64_t ws_floats,
                                      hipStream_t stream) {
  const Q4Cache c{static_cast<uint8_t*>(k_codes), static_cast<_Float16*>(k_meta), static_cast<uint8_t*>(v_codes),
                  static_cast<_Float16*>(v_meta), n_seq, kv_heads, max_len};
  if (const int rc = check_cache("decode_attention_q4", c, head_dim)) return rc;
  if (dtype != FW_F16 && dtype != FW_BF16) return fw_fail(FW_EINVAL, "decode_attention_q4: dtype must be FW_F16 or FW_BF16");
  if (!q || !lens || !out) return fw_fail(FW_EINVAL, "decode_attention_q4: null pointer");
  if (!k_new != !v_new) return fw_fail(FW_EINVAL, "decode_attention_q4: k_new and v_new must be given together");
  if (heads <= 0 || heads % kv_heads) return fw_fail(FW_EINVAL, "decode_attention_q4: heads must be a multiple of kv_heads");
  if (!rows_ok(q, q_row, q_head) || !rows_ok(out, o_row, o_head) || (k_new && (!rows_ok(k_new, k_row, k_head) || !rows_ok(v_new, v_row, v_head))))
    return fw_fail(FW_EINVAL, "decode_attention_q4: q, out, k_new and v_new must be 16-byte aligned with strides in multiples of 8");
  const int64_t need = fw_decode_attention_q4_ws_floats(n_seq, heads, kv_heads, max_len, head_dim);
  if (!ws || ws_floats < need || !aligned(ws, 16))
    return fw_fail(FW_EINVAL, "decode_attention_q4: workspace needs %lld floats, 16-byte aligned", static_cast<long long>(need));
  const Q4Attn a{q, out, q_row, q_head, o_row, o_head, Q4Rows{k_new, v_new, k_row, k_head, v_row, v_head}, lens, c, heads, scale};
  Q4_LAUNCH(decode_attention_q4_kernel, dtype, head_dim, dim3(heads, n_seq), dim3(256), stream, a);
  return fw_check_launch("decode_attention_q4");
}
