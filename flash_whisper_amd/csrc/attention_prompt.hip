// Attention over whole prompts for gfx950: sequences of different lengths packed one after another, query
// heads grouped over key/value heads, causal from the end of the keys or not.
// Built with MFMA results in VGPRs (-mllvm -amdgpu-mfma-vgpr-form), as the encoder attention and for its reason.
#include <type_traits>

#include "lds_pipe.h"
#include "packed_rows.h"

namespace fw {
namespace {

typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef short s4v __attribute__((ext_vector_type(4)));

template <class T>
struct Types;
template <>
struct Types<_Float16> {
  typedef h8v v8;
  typedef h2v v2;
  static constexpr uint32_t kExp = 0x7C007C00u, kExpOne = 0x04000400u;  // a pair's exponent fields, and their last bits
};
template <>
struct Types<__bf16> {
  typedef b8v v8;
  typedef b2v v2;
  static constexpr uint32_t kExp = 0x7F807F80u, kExpOne = 0x00800080u;
};

__device__ __forceinline__ f16v mfma32(const h8v& a, const h8v& b, const f16v& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mfma32(const b8v& a, const b8v& b, const f16v& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float add_pair(h2v x, float s) {
  return __builtin_amdgcn_fdot2(x, h2v{static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)}, s, false);
}
__device__ __forceinline__ float add_pair(b2v x, float s) {
  return __builtin_amdgcn_fdot2_f32_bf16(x, b2v{static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)}, s, false);
}

struct PromptArgs {
  const void *q, *k, *v;
  void* out;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;
  const int64_t *cu_q, *cu_k;
  int64_t q_rows, k_rows;
  int n_seq, heads, kv_heads;
  float scale;
};

// ------------------------------------------------------------------------------------------
// A row of a block is a query and one of the heads that share a key/value head: row i of a sequence is query
// i / group and head i % group, so grouped heads share every key that is staged, and a few queries fill a tile.
// Block = QG waves of 32 rows x KP key parts (TK-key tiles t with t % KP == part); the parts' (m, l, O) are
// merged through LDS at the end. Per tile a wave computes S^T = K Q^T (keys x rows), so that a lane holds scores of
// one row and maximum and sum need one cross-lane step, and feeds P^T from the S^T layout as the B operand of
// O^T = V^T P^T: a lane of half lg = lane / 32 holds keys 4 lg .. 4 lg + 3 and 8 more of every 16.
//  - K and V tiles arrive row-major by direct-to-LDS copies in a ring of ST stages, their 16-byte chunks swizzled:
//    K so that 16 rows' same chunk lies in 16 different bank groups, V so that 4 rows' 64 bytes do.
//  - V^T operands are read with the transposing LDS read: 16 lanes name 4 keys x 16 dims, 8 bytes each, and lane i
//    gets dim i of the 4 keys. Two reads give the 8 keys the lane holds in P^T.
//  - Weights are taken against the maximum so far and only their sum, which is wanted anyway, tells whether a score is far
//    above it: then, and in the first tile, the maximum is looked for and the weights are taken (again) against it. Up to
//    kMost a weight keeps its precision in fp16 as in bf16; a larger one, an infinity for fp16, never reaches a product.
//    Without the maximum in every tile 8192 tokens of 20 heads of 64 take 202 us instead of 212.
//  - Weights are rounded to the type, which the matrix instructions take; their sum, in fp32, is over the rounded ones, so that
//    a common error cancels. Off the values in 64 bits by (rms, relative) 1.74e-4 for 4 causal fp16 tokens, where one rounding
//    of them to fp16 is off by 1.70e-4, 2.02e-4 for ragged ones of up to 4096 (2.02e-4), 1.645e-3 for 8192 in bf16 (1.643e-3).
//  - Masked tiles (the causal diagonal, the last one of a sequence): a masked score is replaced before the maximum,
//    whatever it is. A masked weight of 0 does not undo an infinity or NaN in V, so the block looks for them in
//    the tile, puts zeros there, and keeps for each dim the first key with either infinity and with a NaN: a row sees
//    the keys up to its limit, so at the end it gets those whose first key it sees.
// Bound by the power that the products take for heads of 128 (8192 tokens of 32 heads, causal, bf16: 505 us, 1.09 PFLOP/s,
// where a library product of 8192^3 reaches 1.2; with zeros as inputs 400 us). Heads of 64 have half the products for every
// exponential (8192 tokens of 20 heads: 203 us, 0.85 PFLOP/s: 32 exponentials, 32 fused multiply-adds, 16 conversions and 16
// sums for the 16 products of a wave's tile): no unit is full (12 ragged sequences: vector 45%, matrix 31%, LDS 16% of the
// cycles), and a wave, of which a SIMD has 1.8 on average, waits for 36% of its time, each step of its chain for the one before.
// ------------------------------------------------------------------------------------------
constexpr float kMost = 4096.f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kAhead = 2;  // 1 to 4 measured within 2% of each other

template <int D>
__device__ __forceinline__ int k_slot(int row, int chunk) {
  return D == 64 ? chunk ^ ((row >> 1) & 7) : chunk ^ (row & 15);
}
template <int D>
__device__ __forceinline__ int v_slot(int row, int chunk) {
  return D == 64 ? chunk ^ (((row >> 1) & 1) << 2) : chunk ^ ((row & 3) << 2);
}

// Where a block works: sequence rows [row0, row0 + ROWS) of `rows`, queries from packed row q0, keys from k0.
struct Job {
  int seq, row0, rows, nq, nk;
  int64_t q0, k0;
};

// Query or key rows of sequence s, its starts clamped to the rows there are.
__device__ __forceinline__ int seq_rows(const int64_t* cu, int64_t rows, int s, int64_t& begin) {
  begin = within(cu[s], 0, rows);
  return static_cast<int>(within(cu[s + 1], begin, rows) - begin);
}

// What the block of number `slot` does; false: nothing. Sequence s has the slots from cu_q[s] group / ROWS + s on:
// one more than its rows fill, which its last block may need, and no sum over the sequences before it.
template <int ROWS>
__device__ __forceinline__ bool find_job(const PromptArgs& a, int64_t slot, Job& job) {
  const int group = a.heads / a.kv_heads;
  const auto start = [&](int s) { return within(a.cu_q[s], 0, a.q_rows) * group / ROWS + s; };
  job.seq = last_started(a.n_seq, slot, start);
  if (job.seq < 0) return false;
  job.nq = seq_rows(a.cu_q, a.q_rows, job.seq, job.q0);
  job.nk = seq_rows(a.cu_k, a.k_rows, job.seq, job.k0);
  job.rows = job.nq * group;
  const int64_t row0 = (slot - start(job.seq)) * ROWS;
  job.row0 = static_cast<int>(row0);
  return row0 >= 0 && row0 < job.rows;  // (negative: of starts that do not ascend)
}

template <int D>
struct State {
  f16v o[D / 32];  // O^T blocks of 32 dims; lane (row, lg), register r: dim 8 (r / 4) + 4 lg + r % 4
  float m, l;   // l: this lane's keys only
};

// Byte offsets of a lane's operands in staged tiles, apart from the multiples of 8 and 32 rows that the reads add as
// constants: K row lr, chunk 2 j + lg; V row 4 lg + i / 4, dims 32 db + 16 (lane / 16 % 2) + 4 (i % 4), for i =
// lane % 16. The swizzles do not depend on those multiples.
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) s4v lds_s4;
template <int D>
struct Offsets {
  uint32_t k[D / 16], v[D / 32];
};
template <int D>
__device__ __forceinline__ Offsets<D> lane_offsets(int lane) {
  Offsets<D> o;
  const int lr = lane & 31, lg = lane >> 5, i = lane & 15, row = 4 * lg + (i >> 2);
#pragma unroll
  for (int j = 0; j < D / 16; ++j) o.k[j] = lr * (2 * D) + k_slot<D>(lr, 2 * j + lg) * 16;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
    o.v[db] = row * (2 * D) + v_slot<D>(row, 4 * db + 2 * ((lane >> 4) & 1) + ((i >> 1) & 1)) * 16 + (i & 1) * 8;
  return o;
}

// V^T operand of 32 dims and 16 keys: two transposing reads of 4 keys a lane half, 8 keys apart.
template <class T, int D>
__device__ __forceinline__ typename Types<T>::v8 read_vt(lds_u8* at) {
  const s4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4*>(at));
  const s4v b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4*>(at + 8 * 2 * D));
  return __builtin_bit_cast(typename Types<T>::v8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// The first keys with a value that is no number, by dim: infinities, negative ones, NaNs.
constexpr int kNoKey = 0x7FFFFFFF;
template <int D>
struct OddValues {
  int first[3][D];
  int any;
};

// Looks through 16 bytes of a staged V tile: 8 dims from d of key `key`.
template <class T, int D>
__device__ __forceinline__ void set_aside(uint32_t at, int key, int d, OddValues<D>& odd) {
  typedef __attribute__((address_space(3))) u32x4 lds_u4;
  u32x4 x = *reinterpret_cast<lds_u4*>(static_cast<uintptr_t>(at));
  uint32_t found = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) found |= (x[e] & Types<T>::kExp) + Types<T>::kExpOne;
  if ((found & 0x80008000u) == 0) return;
  typename Types<T>::v8 y = __builtin_bit_cast(typename Types<T>::v8, x);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float f = static_cast<float>(y[e]);
    if (__builtin_fabsf(f) < INFINITY) continue;
    atomicMin(&odd.first[f != f ? 2 : f > 0.f ? 0 : 1][d + e], key);
    y[e] = static_cast<T>(0.f);
  }
  *reinterpret_cast<lds_u4*>(static_cast<uintptr_t>(at)) = __builtin_bit_cast(u32x4, y);
  odd.any = 1;
}

// A wave's tile: K at LDS address k, V at v; keys kv0 .., of which the lane's row sees those up to `limit`; masked:
// some row does not see all of them.
template <class T, int D, int TK>
__device__ __forceinline__ void tile(uint32_t k, uint32_t v, const Offsets<D>& off, const typename Types<T>::v8 (&q)[D / 16],
                                     float factor, int kv0, int limit, bool masked, int lane, State<D>& st) {
  typedef typename Types<T>::v8 v8;
  typedef typename Types<T>::v2 v2;
  const int lg = lane >> 5;
  typedef __attribute__((address_space(3))) v8 lds_v8;
  constexpr int NB = TK / 32, NJ = D / 16, NP = TK / 16, ND = D / 32;
  f16v s[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
  // Operands are read kAhead steps before the products that take them; the scheduling barriers keep it at that,
  // since all of a tile's operands at once do not fit the registers.
  v8 kf[kAhead + 1][NB];
  const auto read_k = [&](int j) {
    lds_u8* at = reinterpret_cast<lds_u8*>(static_cast<uintptr_t>(off.k[j] + k));
#pragma unroll
    for (int b = 0; b < NB; ++b) kf[j % (kAhead + 1)][b] = *reinterpret_cast<lds_v8*>(at + b * (32 * 2 * D));
  };
#pragma unroll
  for (int j = 0; j < kAhead; ++j) read_k(j);
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    if (j + kAhead < NJ) read_k(j + kAhead);
#pragma unroll
    for (int b = 0; b < NB; ++b) s[b] = mfma32(kf[j % (kAhead + 1)][b], q[j], s[b]);
    __builtin_amdgcn_sched_barrier(0);
  }
  v8 vf[2][ND];  // V^T operands: the first step's wait behind the softmax
  lds_u8* vat[ND];
#pragma unroll
  for (int db = 0; db < ND; ++db) vat[db] = reinterpret_cast<lds_u8*>(static_cast<uintptr_t>(off.v[db] + v));
  const auto read_v = [&](int j) {
#pragma unroll
    for (int db = 0; db < ND; ++db) vf[j % 2][db] = read_vt<T, D>(vat[db] + j * (16 * 2 * D));
  };
  read_v(0);
  if (masked) {  // wave-uniform
    const int rel = limit - kv0 - 4 * lg;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (32 * b + 8 * (r >> 2) + (r & 3) > rel) s[b][r] = -INFINITY;
  }
  v8 p[TK / 16];
  float sum;
  // A tile's weights are taken against the maximum so far; where their sum says that a score is far above it (or where
  // a row has seen no key yet), the maximum is looked for and they are taken again.
  for (bool behind = __builtin_amdgcn_ballot_w64(st.m == -INFINITY) != 0;; behind = true) {  // wave-uniform
    if (behind) {
      float top = -INFINITY;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = __builtin_elementwise_maximum(top, s[b][r]);  // a NaN stays, as does the row's
      top = xor_max<32>(top) * factor;
      const float m_new = __builtin_elementwise_maximum(st.m, top);
      const float corr = st.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m - m_new);
      st.l *= corr;
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) st.o[db][r] *= corr;
      st.m = m_new;
    }
    const float m = st.m == -INFINITY ? 0.f : st.m;  // a row that has seen no key yet: its weights are 0
    float part[NB] = {};
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        v2 x;
        x[0] = static_cast<T>(__builtin_amdgcn_exp2f(fmaf(s[b][r], factor, -m)));
        x[1] = static_cast<T>(__builtin_amdgcn_exp2f(fmaf(s[b][r + 1], factor, -m)));
        part[b] = add_pair(x, part[b]);
        p[2 * b + (r >> 3)][r & 7] = x[0];
        p[2 * b + (r >> 3)][(r & 7) + 1] = x[1];
      }
    sum = NB == 1 ? part[0] : part[0] + part[NB - 1];
    if (behind || !__builtin_amdgcn_ballot_w64(sum > kMost)) break;
  }
  st.l += sum;
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    if (j + 1 < NP) read_v(j + 1);
#pragma unroll
    for (int db = 0; db < ND; ++db) st.o[db] = mfma32(vf[j % 2][db], p[j], st.o[db]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <class T, int D, int QG, int KP, int TK, int ST, bool CAUSAL>
__global__ void __launch_bounds__(QG * KP * 64, 2) prompt_attention_kernel(PromptArgs a) {
  typedef typename Types<T>::v8 v8;
  constexpr int kRows = 32 * QG, kTile = TK * D * 2, kStage = KP * 2 * kTile, kChunks = D / 8;
  constexpr int kCopies = kTile / 1024 / QG;  // per wave, of a K tile and of a V tile
  constexpr int kMergeF = 2 + D / 2;          // floats a lane hands over
  static_assert(kTile / 1024 % QG == 0, "copies");
  constexpr int kRing = ST * kStage, kMerge = (KP - 1) * QG * 64 * kMergeF * 4;
  __shared__ __align__(1024) uint8_t ring[kRing > kMerge ? kRing : kMerge];
  __shared__ OddValues<D> odd;

  const int kvh = blockIdx.x % a.kv_heads, group = a.heads / a.kv_heads;
  Job job;
  // causal: from the last rows, whose blocks take longest
  const unsigned slot = blockIdx.x / a.kv_heads, slots = gridDim.x / a.kv_heads;
  if (!find_job<kRows>(a, CAUSAL ? slots - 1 - slot : slot, job)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wq = wave % QG, part = wave / QG, lr = lane & 31, lg = lane >> 5;
  // this lane's row (its last one for lanes past the end, which store nothing) and the last key it sees
  const int row = job.row0 + 32 * wq + lr, at_row = min(row, job.rows - 1), query = at_row / group;
  const int head = kvh * group + at_row % group;
  const int seen0 = CAUSAL ? job.nk - job.nq : job.nk - 1;  // last key that query 0 sees
  const int limit = CAUSAL ? seen0 + query : seen0;
  const auto limit_of = [&](int r) { return CAUSAL ? seen0 + min(r, job.rows - 1) / group : seen0; };
  // (a wave whose rows are all past the end takes part in the copies alone)
  const int wave_row = job.row0 + 32 * wq, wave_first = limit_of(wave_row);
  const int wave_last = wave_row < job.rows ? limit_of(wave_row + 31) : -1;
  const int block_first = limit_of(job.row0), block_last = limit_of(job.row0 + kRows - 1);

  v8 q[D / 16];
  const T* qp = static_cast<const T*>(a.q) + (job.q0 + query) * a.q_row + head * a.q_head + 8 * lg;
#pragma unroll
  for (int j = 0; j < D / 16; ++j) q[j] = *reinterpret_cast<const v8*>(qp + 16 * j);
  if (a.scale < 0.f) {  // scores are scaled by a positive factor after the product
#pragma unroll
    for (int j = 0; j < D / 16; ++j) q[j] = -q[j];
  }
  // 0: the smallest number instead, against which the largest bf16 score, below 2^128, vanishes too; a masked score
  // (-infinity) times zero would be NaN. fp32 keeps subnormal numbers here.
  const float factor = fmaxf(__builtin_fabsf(a.scale) * kLog2e, __FLT_DENORM_MIN__);

  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ring));
  const T* kbase = static_cast<const T*>(a.k) + job.k0 * a.k_row + kvh * a.k_head;
  const T* vbase = static_cast<const T*>(a.v) + job.k0 * a.v_row + kvh * a.v_head;
  const int tiles = block_last < 0 ? 0 : block_last / TK + 1, stages = (tiles + KP - 1) / KP;
  const int crow = lane / kChunks, cslot = lane % kChunks;  // a copy fills 64 / kChunks rows
  const auto issue = [&](int p) {
    // a part whose tile is past the end copies the last one again: every wave issues the same number of copies
    const int t = min(KP * p + part, tiles - 1), kv0 = t * TK, last = job.nk - 1 - kv0;
    const uint32_t stage = lds0 + (p % ST) * kStage + part * 2 * kTile;
    const T *kb = kbase + kv0 * a.k_row, *vb = vbase + kv0 * a.v_row;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int blk = kCopies * wq + i, r = blk * (64 / kChunks) + crow, rc = min(r, last);  // keys past the end: the last one
      dma16_s(static_cast<uint32_t>(rc) * static_cast<uint32_t>(a.k_row * 2) + k_slot<D>(r, cslot) * 16, kb, stage + blk * 1024);
    }
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int blk = kCopies * wq + i, r = blk * (64 / kChunks) + crow, rc = min(r, last);
      dma16_s(static_cast<uint32_t>(rc) * static_cast<uint32_t>(a.v_row * 2) + v_slot<D>(r, cslot) * 16, vb,
              stage + kTile + blk * 1024);
    }
  };
#pragma unroll
  for (int p = 0; p < ST - 1; ++p)
    if (p < stages) issue(p);

  const Offsets<D> off = lane_offsets<D>(lane);
  State<D> st;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) st.o[db][r] = 0.f;
  st.m = -INFINITY;
  st.l = 0.f;
  for (int i = tid; i < 3 * D; i += QG * KP * 64) (&odd.first[0][0])[i] = kNoKey;
  if (tid == 0) odd.any = 0;

  // Waves of a part share its tiles; with one wave a part the rings are the waves' own and nobody waits for others.
  const auto sync = [&] {
    if constexpr (QG > 1) lds_barrier();
    else lds_reads_done();
  };
  if constexpr (QG == 1) lds_barrier();  // `odd` is cleared
  for (int p = 0; p < stages; ++p) {
    // stage p visible to every wave of the part, every one done with stage p - 1, whose slot takes stage p + ST - 1
    if constexpr (ST > 1) {
      wait_stages_ahead<2 * kCopies, ST - 1>(min(ST - 2, stages - 1 - p));
      sync();
      if (p + ST - 1 < stages) issue(p + ST - 1);
    } else {
      sync();
      issue(p);
      wait_vmcnt<0>();
      sync();
    }
    const int t = KP * p + part, kv0 = t * TK;
    const uint32_t k = lds0 + (p % ST) * kStage + part * 2 * kTile, v = k + kTile;
    if (KP * (p + 1) * TK - 1 > block_first) {  // some row of the block sees only a part of this stage
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int blk = kCopies * wq + i, r = blk * (64 / kChunks) + crow;
        set_aside<T, D>(v + blk * 1024 + lane * 16, kv0 + r, v_slot<D>(r, cslot) * 8, odd);
      }
      sync();
    }
    if (kv0 <= wave_last) tile<T, D, TK>(k, v, off, q, factor, kv0, limit, kv0 + TK - 1 > wave_first, lane, st);
  }

  st.l = xor_add<32>(st.l);
  float m = st.m, l = st.l, scale_o = 1.f;
  if constexpr (KP > 1) {
    // parts 1 .. KP - 1 hand (m, l, O) through LDS to the wave of part 0 with the same rows
    lds_barrier();  // every wave is done with the ring
    float* mine = reinterpret_cast<float*>(ring) + (wq * 64 + lane) * kMergeF;
    constexpr int kPartF = QG * 64 * kMergeF;
    if (part > 0) {
      float* to = mine + (part - 1) * kPartF;
      to[0] = st.m;
      to[1] = st.l;
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) to[2 + 16 * db + r] = st.o[db][r];
    }
    lds_barrier();
    if (part > 0) return;
#pragma unroll
    for (int i = 0; i < KP - 1; ++i) m = fmaxf(m, mine[i * kPartF]);
    scale_o = st.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m - m);
    l *= scale_o;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) st.o[db][r] *= scale_o;
#pragma unroll
    for (int i = 0; i < KP - 1; ++i) {
      const float* from = mine + i * kPartF;
      const float e = from[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(from[0] - m);
      l = fmaf(e, from[1], l);
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) st.o[db][r] = fmaf(e, from[2 + 16 * db + r], st.o[db][r]);
    }
  }
  else {
    lds_barrier();  // `odd` is complete and visible
  }
  if (row >= job.rows) return;
  if (odd.any) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int d = 32 * db + 8 * (r >> 2) + 4 * lg + (r & 3);
        if (odd.first[0][d] <= limit) st.o[db][r] += INFINITY;
        if (odd.first[1][d] <= limit) st.o[db][r] -= INFINITY;
        if (odd.first[2][d] <= limit) st.o[db][r] = __builtin_nanf("");
      }
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;  // no key seen: zeros
  T* op = static_cast<T*>(a.out) + (job.q0 + query) * a.o_row + head * a.o_head + 4 * lg;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      typedef T v4 __attribute__((ext_vector_type(4)));
      v4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = static_cast<T>(st.o[db][4 * j + e] * inv);
      *reinterpret_cast<v4*>(op + 32 * db + 8 * j) = x;
    }
}

constexpr int kCus = 256;

// How a call shares out its rows, FW_PROMPT_*.
// Blocks of 128 rows stage every tile for four waves and are the fastest where they fill the CUs. Few rows over many
// keys are given to several waves, whose parts of the keys are merged: 8 parts while blocks of 32 rows have a CU
// each, 2 parts of 64 keys while blocks of 64 rows are at most two a CU (causal ones of heads of 64, which end at
// different times and of which a CU holds two, four); then, and where the keys are few, 2 parts of
// 32 keys, up to 1.5 blocks of 128 rows a CU (2 where the keys are few and a block is over soon). Where the keys are a
// tile a sequence, a wave works alone and many blocks share a CU. Keys a sequence are the average of all rows there are,
// behind the last sequence too, since only the device has the lengths: one long prompt among many of a token runs in single waves (63 x 1 token and 1900 x 20 heads of 64
// 48 us, the 1900 alone 22.5; 255 x 1 and 4096 122 and 67), where 2000 prompts of 8 tokens are three times as fast.
// us of 128 rows / 64 rows, 2 parts of 32 keys / of 64 keys / 32 rows, 8 parts:
//   heads of 64, 1 x 4 queries x 20 heads over 1500 keys 20.7 / 18.5 / 14.1 / 11.3; 6 x 4 likewise 21.7 / 19.5 / 15.3 /
//   13.5; 1 x 500 x 20, causal 11.1 / 9.4 / 8.3 / 10.9; 1 x 2000 x 20 30.9 / 26.9 / 22.6 / 38.5; 2 x 1500 x 20 31.2 / 29.3 /
//   27.3 / 49.7; 3 x 1500 x 20 41.1 /
//   39.8 / 40.2 / 72.5; 1 x 8192 x 20 204 / 257 / 234 / 386; 16 x 4 .. 224 x 20 9.4 / 8.3 / 11.5 / 20; over 1500
//   keys 35.9 / 39.4 / 46.5 / 57;
//   heads of 128 over 8 key/value heads, 4 x 32 x 32 over 4000 keys 86 / 72 / 57 / 33; 8 x 64 x 32 likewise 114 / 102 / 82 /
//   88; 1 x 1000 x 32, causal 27.1 / 23.9 / 26.2 / 47.4; 1 x 4096 x 32 157 / 183 / 224 / 314.
// Heads of 64, 128 rows / the single wave: 1 x 4 x 20 4.4 / 4.0; 2000 x 8 x 20 246 / 84; 64 x 64 x 20 14.9 / 13.9; 64 x 1
// .. 200 x 8 over 2 heads 7.0 / 8.5.
// (8 parts with a second stage where the LDS holds it: 1 x 4 queries x 20 heads over 1500 keys 11.3 us against 12.1, 5 x 8
// x 20 over 2705 16.5 against 17.7.)
int prompt_form(int n_seq, int64_t rows, int64_t k_rows, int kv_heads, int dim, bool causal) {
  const int64_t keys = k_rows / n_seq;
  const auto blocks_of = [&](int64_t n) { return (rows / n + n_seq) * kv_heads; };
  if (blocks_of(32) <= kCus && keys >= 512) return FW_PROMPT_8_PARTS;
  if (keys <= 32) return FW_PROMPT_WAVES;
  if (blocks_of(64) <= (causal && dim == 64 ? 4 : 2) * kCus && keys >= 384) return FW_PROMPT_2_PARTS;
  if (blocks_of(128) <= (keys < 256 ? 2 * kCus : kCus * 3 / 2)) return FW_PROMPT_2_SHORT_PARTS;
  return FW_PROMPT_128_ROWS;
}

// What a call asks of its sizes; FW_OK or FW_EINVAL.
int check_sizes(int n_seq, int64_t q_rows, int64_t k_rows, int heads, int kv_heads, int head_dim) {
  if (n_seq <= 0 || q_rows < 0 || k_rows < 0)
    return fw_fail(FW_EINVAL, "prompt_attention: n_seq must be positive, rows not negative");
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads)
    return fw_fail(FW_EINVAL, "prompt_attention: heads must be a multiple of kv_heads");
  if (head_dim != 64 && head_dim != 128) return fw_fail(FW_EINVAL, "prompt_attention: head_dim must be 64 or 128");
  // rows x heads of a sequence are counted in 32 bits
  if (q_rows > 0x7FFFFF00 / (heads / kv_heads) || k_rows > 0x7FFFFF00) return fw_fail(FW_EINVAL, "prompt_attention: too many rows");
  return FW_OK;
}

bool rows_ok(const void* p, int64_t row, int64_t head) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && row % 8 == 0 && head % 8 == 0;
}

}  // namespace
}  // namespace fw

using namespace fw;

extern "C" int fw_prompt_attention_form(int n_seq, int64_t q_rows, int64_t k_rows, int heads, int kv_heads, int head_dim,
                                        int causal) {
  if (const int rc = check_sizes(n_seq, q_rows, k_rows, heads, kv_heads, head_dim)) return rc;
  return prompt_form(n_seq, q_rows * (heads / kv_heads), k_rows, kv_heads, head_dim, causal);
}

extern "C" int fw_prompt_attention(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                                   const void* v, int64_t v_row, int64_t v_head, void* out, int64_t o_row, int64_t o_head,
                                   const int64_t* cu_q, const int64_t* cu_k, int n_seq, int64_t q_rows, int64_t k_rows,
                                   int heads, int kv_heads, int head_dim, int dtype, float scale, int causal,
                                   hipStream_t stream) {
  if (const int rc = check_sizes(n_seq, q_rows, k_rows, heads, kv_heads, head_dim)) return rc;
  if (dtype != FW_F16 && dtype != FW_BF16) return fw_fail(FW_EINVAL, "prompt_attention: dtype must be FW_F16 or FW_BF16");
  if (!cu_q || !cu_k || (q_rows > 0 && (!q || !out)) || (k_rows > 0 && (!k || !v)))
    return fw_fail(FW_EINVAL, "prompt_attention: null pointer");
  if ((q_rows > 0 && (!rows_ok(q, q_row, q_head) || !rows_ok(out, o_row, o_head))) ||
      (k_rows > 0 && (!rows_ok(k, k_row, k_head) || !rows_ok(v, v_row, v_head))))
    return fw_fail(FW_EINVAL, "prompt_attention: q, k, v and out must be 16-byte aligned with strides in multiples of 8");
  if (!(__builtin_fabsf(scale) * kLog2e < INFINITY))
    return fw_fail(FW_EINVAL, "prompt_attention: scale must be finite (and below 2.3e38 in size)");
  // 64 rows of k and of v within the copies' 32-bit byte offsets
  if (k_row < 0 || v_row < 0 || k_row >= (1 << 25) || v_row >= (1 << 25))
    return fw_fail(FW_EINVAL, "prompt_attention: row strides of k and v must be below 2^25 elements");
  if (q_rows == 0) return FW_OK;
  const PromptArgs a{q, k, v, out, q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head, cu_q, cu_k,
                     q_rows, k_rows, n_seq, heads, kv_heads, scale};
  const int64_t rows = q_rows * (heads / kv_heads);
  const int form = prompt_form(n_seq, rows, k_rows, kv_heads, head_dim, causal);
  int rc = FW_OK;
  const auto launch = [&](auto kernel, int per_block, int threads) {
    const int64_t blocks = (rows / per_block + n_seq) * kv_heads;  // a sequence's last block may be partial
    if (!grid_ok(blocks, threads)) rc = fw_fail(FW_EINVAL, "prompt_attention: too many rows");
    else hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(threads), 0, stream, a);
  };
  const auto by_rows = [&](auto t, auto d, auto mask) {
    typedef decltype(t) T;
    constexpr int D = decltype(d)::value;
    constexpr bool M = decltype(mask)::value;
    switch (form) {
      case FW_PROMPT_8_PARTS: launch(prompt_attention_kernel<T, D, 1, 8, 32, D == 64 ? 2 : 1, M>, 32, 512); break;
      case FW_PROMPT_WAVES: launch(prompt_attention_kernel<T, D, 1, 1, 32, 1, M>, 32, 64); break;
      case FW_PROMPT_2_PARTS: launch(prompt_attention_kernel<T, D, 2, 2, 64, 2, M>, 64, 256); break;
      case FW_PROMPT_2_SHORT_PARTS: launch(prompt_attention_kernel<T, D, 2, 2, 32, 2, M>, 64, 256); break;
      default: launch(prompt_attention_kernel<T, D, 4, 1, 64, 2, M>, 128, 256);
    }
  };
  const auto by_mask = [&](auto t, auto d) { causal ? by_rows(t, d, std::true_type()) : by_rows(t, d, std::false_type()); };
  const std::integral_constant<int, 64> d64;
  const std::integral_constant<int, 128> d128;
  if (dtype == FW_F16) head_dim == 64 ? by_mask(_Float16(), d64) : by_mask(_Float16(), d128);
  else head_dim == 64 ? by_mask(__bf16(), d64) : by_mask(__bf16(), d128);
  return rc ? rc : fw_check_launch("prompt_attention");
}
