// Key/value cache held in 4 bits for gfx950: rows written into it, read back, and the single-token
// attention over it. Layout (L = max_len, a multiple of 32; D = 64 or 128; 32 dims of a row, a group,
// share a step and a low value):
//   k_codes [seq][head][L][D / 2]          row-major: lane = key of the score products
//   k_meta  [seq][head][L][D / 32] {step, low}
//   v_codes [seq][head][L / 8][D / 4][16]  8 rows x 4 dims in 16 bytes, row t's 4 dims at byte 2 (t % 8):
//                                          one 16-byte load holds a lane's 8 keys of the P V products
//   v_meta  [seq][head][L / 8][D / 32] {step of 8 rows, low of 8 rows}
// A code c stands for fp16(low + step c), one rounding; 5 bits a value with step and low.
#include <algorithm>
#include <type_traits>

#include "packed_rows.h"

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
// Waits for this wave's LDS accesses; none moves across it.
__device__ __forceinline__ void lds_wave_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

struct Q4Slot {
  int seq;        // -1: nothing to do
  int64_t first;  // packed row of cache row `row` (may lie before the sequence's own rows)
  int64_t begin, end;  // the sequence's packed rows
  int64_t row;    // first cache row of the block, a multiple of 8 (may be negative or past the cache)
};

__device__ __forceinline__ Q4Slot q4_slot(const int64_t* cu, const int64_t* pos, int n_seq, int64_t rows, int64_t slot) {
  Q4Slot r{-1, 0, 0, 0, 0};
  r.seq = last_started(n_seq, slot, [&](int s) { return within(cu[s], 0, rows) / 8 + 2 * static_cast<int64_t>(s); });
  if (r.seq < 0) return r;
  r.begin = within(cu[r.seq], 0, rows);
  r.end = within(cu[r.seq + 1], r.begin, rows);
  const int64_t p = pos[r.seq], block = slot - (r.begin / 8 + 2 * static_cast<int64_t>(r.seq));
  r.row = (p & ~int64_t{7}) + 8 * block;
  r.first = r.begin + (r.row - p);
  if (r.first >= r.end) r.seq = -1;
  return r;
}

// A group's step and low from its smallest and largest value: the step rounded towards zero, so that
// low + 15 step stays within the group's values and no finite value reads back as an infinity. A group
// holding a NaN, an infinity or a bf16 value that fp16 rounds to one gets a NaN step and reads back as NaN.
constexpr float kPastHalf = 65520.f;
__device__ __forceinline__ void q4_meta(float lo, float hi, bool finite, _Float16& step, _Float16& low) {
  const auto rtz = __builtin_amdgcn_cvt_pkrtz((hi - lo) * (1.0f / 15.0f), 0.f);
  step = finite ? static_cast<_Float16>(rtz[0]) : static_cast<_Float16>(__builtin_nanf(""));
  low = f2h(lo);
}

// 8 values of a lane to 8 codes in a dword, element e in bits 4 e; the 4 lanes of a group agree on its meta. The
// quotient (x - low) / step: a product by the reciprocal (itself correctly rounded) and one correction by the
// remainder give the correctly rounded one, so ties go to the even code.
template <class T>
__device__ __forceinline__ uint32_t q4_pack8(const typename Vec8<T>::type& x, _Float16& step, _Float16& low) {
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = static_cast<float>(x[e]);
  float lo = f[0], hi = f[0];  // a NaN makes both NaN
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    lo = __builtin_elementwise_minimum(lo, f[e]);
    hi = __builtin_elementwise_maximum(hi, f[e]);
  }
  lo = __builtin_elementwise_minimum(lo, xor_lane<1>(lo));
  hi = __builtin_elementwise_maximum(hi, xor_lane<1>(hi));
  lo = __builtin_elementwise_minimum(lo, xor_lane<2>(lo));
  hi = __builtin_elementwise_maximum(hi, xor_lane<2>(hi));
  q4_meta(lo, hi, lo > -kPastHalf && hi < kPastHalf, step, low);
  const float s = h2f(step), l = h2f(low), inverse = 1.0f / s;
  uint32_t codes = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float d = f[e] - l, q = d * inverse, c = rintf(fmaf(fmaf(-q, s, d), inverse, q));
    codes |= static_cast<uint32_t>(__builtin_amdgcn_fmed3f(c, 0.f, 15.f)) << (4 * e);
  }
  return s > 0.f ? codes : 0u;  // 0 for a group of one value, and for one that is no number
}

// ------------------------------------------------------------------------------------------
// Append: a wave = 8 cache rows x 64 dims of a head (lane = row lane / 8, dims 8 (lane % 8)), K and V. Bound
// by memory: 2 bytes a value in, 0.625 out. K leaves as one dword a lane (whole rows); V's 2-byte
// pieces of 8 rows meet in LDS and leave as one dword a lane where all 8 rows are written, and piece by
// piece at a sequence's ends, where the other rows of the unit stay as they are. 8 x 1500 rows of 20 heads of 64
// (81 MB): 19.9 us, 4.1 TB/s (a large copy reaches 4.7).
// ------------------------------------------------------------------------------------------
template <class T, int D>
__global__ void __launch_bounds__(256) kv_q4_append_kernel(const int64_t* __restrict__ cu,
                                                           const int64_t* __restrict__ pos, int64_t rows, int64_t slots,
                                                           int n_seq, int heads, Q4Rows in, Q4Cache c) {
  __shared__ __align__(16) u16 pieces[4][16][8];
  constexpr int kHalves = D / 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + wave, slot = unit / (heads * kHalves);
  const int part = static_cast<int>(unit % (heads * kHalves)), head = part / kHalves, d0 = part % kHalves * 64;
  if (slot >= slots) return;  // no block barrier below
  const Q4Slot w = q4_slot(cu, pos, n_seq, rows, slot);
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
  const int64_t hr = (static_cast<int64_t>(w.seq) * heads + head) * c.max_len;  // the head's first row
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
    lds_wave_done();
    reinterpret_cast<uint32_t*>(vu)[lane] = reinterpret_cast<const uint32_t*>(&p[0][0])[lane];
  } else if (live) {
    *reinterpret_cast<u16*>(vu + (2 * (lane & 7)) * 16 + 2 * r) = static_cast<u16>(vc);
    *reinterpret_cast<u16*>(vu + (2 * (lane & 7) + 1) * 16 + 2 * r) = static_cast<u16>(vc >> 16);
  }
}

// ------------------------------------------------------------------------------------------
// Read: the rows that an append of the same cu and pos wrote, as the values that they stand for. Waves and
// lanes as in the append, up to P (head, half)s a wave; rows outside the cache read as zeros. The 81 MB of the
// append's example: 13.6 us, part of what the append just wrote coming from the last-level cache.
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

template <class T, int D, int P>
__global__ void __launch_bounds__(256) kv_q4_read_kernel(const int64_t* __restrict__ cu,
                                                         const int64_t* __restrict__ pos, int64_t rows, int64_t slots,
                                                         int n_seq, int heads, Q4Rows out, Q4Cache c) {
  constexpr int kHalves = D / 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  const int parts = heads * kHalves, runs = (parts + P - 1) / P;  // a wave has up to P consecutive (head, half)s of a slot
  const int first = static_cast<int>(unit % runs) * P, count = min(P, parts - first);
  const int64_t slot = unit / runs;
  if (slot >= slots) return;
  const Q4Slot w = q4_slot(cu, pos, n_seq, rows, slot);
  if (w.seq < 0) return;
  const int r = lane >> 3;
  const int64_t token = w.first + r, row = w.row + r;
  if (token < w.begin || token >= w.end) return;
  const bool held = row >= 0 && row < c.max_len;
  uint32_t kc[P], vc[P];
  h2v km[P];
  _Float16 vs[P], vl[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int head = (first + i) / kHalves, d = (first + i) % kHalves * 64 + 8 * (lane & 7);
    kc[i] = vc[i] = 0;
    km[i] = h2v{};
    vs[i] = vl[i] = static_cast<_Float16>(0.f);
    if (!held || i >= count) continue;
    const int64_t hr = (static_cast<int64_t>(w.seq) * heads + head) * c.max_len, at = hr + row, block = (hr + w.row) / 8;
    km[i] = *reinterpret_cast<const h2v*>(c.k_meta + (at * (D / 32) + d / 32) * 2);
    kc[i] = *reinterpret_cast<const uint32_t*>(c.k_codes + at * (D / 2) + d / 2);
    const uint8_t* vu = c.v_codes + (block * (D / 4) + d / 4) * 16 + 2 * r;
    vc[i] = *reinterpret_cast<const u16*>(vu) | static_cast<uint32_t>(*reinterpret_cast<const u16*>(vu + 16)) << 16;
    const _Float16* vm = c.v_meta + (block * (D / 32) + d / 32) * 16;
    vs[i] = vm[r];
    vl[i] = vm[8 + r];
  }
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if (i >= count) break;
    const int head = (first + i) / kHalves, d = (first + i) % kHalves * 64 + 8 * (lane & 7);
    T* ko = static_cast<T*>(const_cast<void*>(out.k)) + token * out.k_row + head * out.k_head + d;
    T* vo = static_cast<T*>(const_cast<void*>(out.v)) + token * out.v_row + head * out.v_head + d;
    *reinterpret_cast<typename Vec8<T>::type*>(ko) = q4_values8<T>(kc[i], km[i][0], km[i][1]);
    *reinterpret_cast<typename Vec8<T>::type*>(vo) = q4_values8<T>(vc[i], vs[i], vl[i]);
  }
}

// ------------------------------------------------------------------------------------------
// Single-token attention. An item is a sequence, a key/value head and up to 16 of the query heads that read it;
// S^T = K Q^T and O^T = V^T P^T are MFMAs of 16 keys or head dims by 16 query heads, so grouped heads share
// every row that is read and dequantised. A wave takes 32 keys at a time.
//  - The scores' rows are assigned to keys so that lane group g = lane / 16 ends with the scores of keys
//    8 g .. 8 g + 7 for query head lane % 16: row i of the first 16 is key 8 (i / 4) + i % 4, of the second 4
//    more. These are the keys of one 16-byte unit of V, which the lane loads as the PV operand's source, so
//    neither scores nor values cross lanes.
//  - Codes become fp16 by or-ing them into 1024's mantissa (1024 + c), subtracting 1024, and one packed fma with
//    step and low, which rounds once as the cache's definition does. Q's dims are permuted to the order in
//    which masking a dword's nibbles yields pairs (0 4, 1 5, 2 6, 3 7).
//  - The running maximum only moves when a score passes it by kSlack (log2 units), so weights are at most 2^8. They are
//    rounded to fp16 for bf16 callers too: the values are fp16, one matrix instruction takes both, and 2^-11 of a weight is
//    an eighth of what a bf16 output is rounded by (64 ragged sequences x 32 heads of 128, bf16: 1.656e-3 rms off the values in 64
//    bits, rounding those to bf16 1.655e-3). Their sum, in fp32, is over the rounded ones, as the products are.
// Bound by memory where the lengths are alike (64 x 8000 keys x 8 heads of 128, 32 query heads: 131 us, 5.0 TB/s with
// what the last-level cache gives; one of 131000: 43 us, 3.9 TB/s), by the longest block and the two launches' latency
// where they are not (64 of 1 to 8000: 28.6 us, 3.0 TB/s), and by latency where there is little to read (300 keys x 20
// heads: 4.8 us). Beside the loads the conversion of the codes takes most: 13 instructions for 8 codes.
// A block takes a chunk of an item's keys; an item of one chunk is finished by its block, the chunks of a longer one
// leave (m, l, O) in the workspace for the combine launch. Only the device knows the lengths: every block works out the
// same chunk from them and finds its piece of work (q4_share, q4_piece); blocks without keys end at once.
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
  int chunk, most;  // keys of the largest chunk, the most chunks of a sequence
  int unit;         // what chunks are multiples of; 0: all have the largest's size
  int pieces;       // pieces of work per item number; 0: an item is one
  float* ws;        // O [pieces][items][cols][D], then (m, l) [pieces][items][cols][2]
};

constexpr int kTileKeys = 32;
constexpr int kCols = 16;  // query heads of an item
constexpr float kSlack = 8.f;
constexpr float kLog2e = 1.4426950408889634f;

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

// A tile's data as loaded: K codes and meta of the lane's two keys, V codes and meta of its 8 keys.
template <int D>
struct Q4Tile {
  uint32_t k[2][D / 32];
  h2v km[2];
  u32x4 v[D / 64];
  h8v vs[D / 64], vl[D / 64];
};

// Where a lane's data of the item's first tile lie; a tile later is kTileKeys rows on.
struct Q4Base {
  const uint8_t *k, *v;
  const _Float16 *km, *vm;
};

template <int D>
__device__ __forceinline__ Q4Base q4_base(const Q4Cache& c, int64_t hr, int lane) {
  const int i = lane & 15, g = lane >> 4;
  const int64_t row = hr + 8 * (i >> 2) + (i & 3), block = hr / 8 + g;
  return Q4Base{c.k_codes + row * (D / 2) + g * (D / 8), c.v_codes + (block * (D / 4) + i) * 16,
                c.k_meta + (row * (D / 32) + g * (D / 32) / 4) * 2, c.v_meta + (block * (D / 32) + i / 8) * 16};
}

template <int D>
__device__ __forceinline__ void q4_load_k(const Q4Base& b, int tile, Q4Tile<D>& t) {
  const int64_t row = static_cast<int64_t>(tile) * kTileKeys;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint8_t* k = b.k + (row + 4 * s) * (D / 2);
    if constexpr (D == 128) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(k);
#pragma unroll
      for (int j = 0; j < 4; ++j) t.k[s][j] = x[j];
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(k);
      t.k[s][0] = x.x;
      t.k[s][1] = x.y;
    }
    t.km[s] = *reinterpret_cast<const h2v*>(b.km + (row + 4 * s) * (D / 32) * 2);
  }
}
template <int D>
__device__ __forceinline__ void q4_load_v(const Q4Base& b, int tile, Q4Tile<D>& t) {
  const int64_t row = static_cast<int64_t>(tile) * kTileKeys;
#pragma unroll
  for (int h = 0; h < D / 64; ++h) {
    t.v[h] = *reinterpret_cast<const u32x4*>(b.v + (row / 8 * (D / 4) + 16 * h) * 16);
    const h8v* m = reinterpret_cast<const h8v*>(b.vm + (row / 8 * (D / 32) + 2 * h) * 16);
    t.vs[h] = m[0];
    t.vl[h] = m[1];
  }
}

// The fresh row of a head, quantised by the wave that has its tile: lanes 0 .. D / 8 - 1 take 8 dims of K each, lanes
// 32 .. 32 + D / 8 - 1 of V. They write it to the cache, and the lanes that hold its place in the tile take it over
// from them: nobody waits for the store, or reads it back.
template <class T, int D>
__device__ __forceinline__ typename Vec8<T>::type q4_fresh_values(const Q4Attn& a, int seq, int kvh, int lane) {
  const T* src = lane < 32 ? static_cast<const T*>(a.fresh.k) + seq * a.fresh.k_row + kvh * a.fresh.k_head
                           : static_cast<const T*>(a.fresh.v) + seq * a.fresh.v_row + kvh * a.fresh.v_head;
  return *reinterpret_cast<const typename Vec8<T>::type*>(src + 8 * (lane & (D / 8 - 1)));
}
template <class T, int D>
__device__ __forceinline__ void q4_fresh(const Q4Attn& a, const typename Vec8<T>::type& values, int64_t hr, int row, int lane,
                                         Q4Tile<D>& t) {
  const Q4Cache& c = a.c;
  const int d = 8 * (lane & (D / 8 - 1)), i = lane & 15, g = lane >> 4;
  _Float16 step, low;
  const uint32_t codes = q4_pack8<T>(values, step, low);
  const h2v meta{step, low};
  if ((lane & 31) < D / 8) {
    if (lane < 32) {
      *reinterpret_cast<uint32_t*>(c.k_codes + (hr + row) * (D / 2) + d / 2) = codes;
      if ((lane & 3) == 0) *reinterpret_cast<h2v*>(c.k_meta + ((hr + row) * (D / 32) + d / 32) * 2) = meta;
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
  const int at = row & (kTileKeys - 1), in_group = at & 7;  // of lane group at / 8; of its 8 keys
  const int word = __builtin_bit_cast(int, meta);
#pragma unroll
  for (int s = 0; s < 2; ++s) {  // K: lane i holds key 8 (i / 4) + 4 s + i % 4
    const bool mine = 8 * (i >> 2) + 4 * s + (i & 3) == at;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint32_t x = __shfl(static_cast<int>(codes), D / 32 * g + j);
      t.k[s][j] = mine ? x : t.k[s][j];
    }
    const int m = __shfl(word, 4 * (g * (D / 32) / 4));
    if (mine) t.km[s] = __builtin_bit_cast(h2v, m);
  }
#pragma unroll
  for (int h = 0; h < D / 64; ++h) {  // V: lane group g holds keys 8 g .., lane i dims 4 i .. of each half
    const uint32_t x = static_cast<uint32_t>(__shfl(static_cast<int>(codes), 32 + 8 * h + i / 2)) >> (16 * (i & 1));
    const h2v m = __builtin_bit_cast(h2v, __shfl(word, 32 + 8 * h + 4 * (i / 8)));
    const bool mine = g == at / 8;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (mine && in_group == 2 * w) t.v[h][w] = (t.v[h][w] & 0xFFFF0000u) | (x & 0xFFFFu);
      if (mine && in_group == 2 * w + 1) t.v[h][w] = (t.v[h][w] & 0xFFFFu) | x << 16;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (mine && in_group == e) {
        t.vs[h][e] = m[0];
        t.vl[h][e] = m[1];
      }
  }
}

// The 4-bit fields at bits 0 (j = 0) or 4 (j = 1) of both halves of u as fp16, then low + step c. Or-ed into the
// mantissa of 1024 a field at bit 0 counts ones, into that of 64 one at bit 4 does: subtracting that leaves c, and
// only the upper byte of a half needs a shift. Mask and exponent are hidden from constant folding, which keeps the
// mask in a scalar register and the exponent in a vector one: v_and_or_b32 takes them so, and no two literals.
// (The instruction itself cannot stand in an asm: the compiler then leaves out the waits that a write to
// registers of an unfinished MFMA needs.)
template <int J>
__device__ __forceinline__ h2v q4_pair(uint32_t u, h2v step, h2v low) {
  uint32_t mask = J ? 0x00F000F0u : 0x000F000Fu, one = J ? 0x54005400u : 0x64006400u;
  asm("" : "+s"(mask));
  asm("" : "+v"(one));
  const h2v c = __builtin_bit_cast(h2v, (u & mask) | one) - static_cast<_Float16>(J ? 64.f : 1024.f);
  return __builtin_elementwise_fma(c, step, low);
}

template <int D>
struct Q4State {
  f4v o[D / 64][4];  // O^T: [64-dim half][dim % 4], lane (h, g), register r: dim 16 g + 4 r + dim % 4
  float m, l;        // l: this lane's keys only
};

// Scores of a tile's keys.
template <int D>
__device__ __forceinline__ void q4_scores(const Q4Tile<D>& t, const h8v (&q)[D / 32], f4v (&s)[2]) {
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    s[kt] = f4v{0.f, 0.f, 0.f, 0.f};
    const h2v step = h2v{t.km[kt][0], t.km[kt][0]}, low = h2v{t.km[kt][1], t.km[kt][1]};
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      h8v k;
      const uint32_t u = t.k[kt][j];
      const h2v x[4] = {q4_pair<0>(u, step, low), q4_pair<1>(u, step, low), q4_pair<0>(u >> 8, step, low),
                        q4_pair<1>(u >> 8, step, low)};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        k[2 * e] = x[e][0];
        k[2 * e + 1] = x[e][1];
      }
      s[kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[j], s[kt], 0, 0, 0);
    }
  }
}

// Their weights and the sum over the values; kTail: only the first `left` keys of the tile count.
template <int D, bool kTail>
__device__ __forceinline__ void q4_values(const Q4Tile<D>& t, f4v (&s)[2], float factor, int left, int lane, Q4State<D>& st) {
  const int g = lane >> 4;
  float top = -INFINITY;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int r = 0; r < 4; r += 2) {
      if constexpr (kTail) {
        if (8 * g + 4 * kt + r >= left) s[kt][r] = -INFINITY;
        if (8 * g + 4 * kt + r + 1 >= left) s[kt][r + 1] = -INFINITY;
      }
      // (a NaN score stays one: its row is NaN anyway; fmaxf would quiet every operand first)
      top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, s[kt][r]), s[kt][r + 1]);
    }
  top = xor_max<32>(xor_max<16>(top)) * factor;
  if (__builtin_amdgcn_ballot_w64(top > st.m + kSlack)) {
    const float m_new = fmaxf(st.m, top), corr = __builtin_amdgcn_exp2f(st.m - m_new);
    st.l *= corr;
#pragma unroll
    for (int h = 0; h < D / 64; ++h)
#pragma unroll
      for (int j = 0; j < 4; ++j) st.o[h][j] *= corr;
    st.m = m_new;
  }
  h8v p;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int r = 0; r < 4; r += 2) {
      h2v x;
      x[0] = f2h(__builtin_amdgcn_exp2f(fmaf(s[kt][r], factor, -st.m)));
      x[1] = f2h(__builtin_amdgcn_exp2f(fmaf(s[kt][r + 1], factor, -st.m)));
      st.l = __builtin_amdgcn_fdot2(x, h2v{static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)}, st.l, false);
      p[4 * kt + r] = x[0];
      p[4 * kt + r + 1] = x[1];
    }
#pragma unroll
  for (int h = 0; h < D / 64; ++h) {
    h8v vs = t.vs[h], vl = t.vl[h];
    if constexpr (kTail) {  // whatever the rows past the end hold, their values count as zeros
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * g + e >= left) vs[e] = vl[e] = static_cast<_Float16>(0.f);
    }
    h8v v[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const h2v step{vs[2 * w], vs[2 * w + 1]}, low{vl[2 * w], vl[2 * w + 1]};
      const uint32_t u = t.v[h][w];
      const h2v x[4] = {q4_pair<0>(u, step, low), q4_pair<1>(u, step, low), q4_pair<0>(u >> 8, step, low),
                        q4_pair<1>(u >> 8, step, low)};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j][2 * w] = x[j][0];
        v[j][2 * w + 1] = x[j][1];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) st.o[h][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[j], p, st.o[h][j], 0, 0, 0);
  }
}

// The item's queries as the products' operand, lane (h, g): dims D / 4 g + 8 j .. in the order of q4_pair's
// pairs, and the factor from raw scores to log2 units. A bf16 query is scaled by a power of two to fit fp16 (its
// 8 bits do down to 2^-17 of the largest element; what is lost below is at most 2^-25 of it); the factor undoes it. A
// negative scale negates the query, a zero one becomes so small that scores vanish. The factor of the scaled query is kept a positive number: against one of
// zero a masked score (-infinity), against an infinite one a score of zero would be NaN. (Raised to 1e-30, scores, of at most
// 2^39, vanish all the same; lowered to the largest number, every score but zero is past 2^79, which fp32 does not resolve.)
template <class T, int D>
struct Q4Query {
  typename Vec8<T>::type x[D / 32];
};
template <class T, int D>
__device__ __forceinline__ Q4Query<T, D> q4_load_query(const Q4Attn& a, int seq, int head, bool live, int lane) {
  Q4Query<T, D> r = {};
  const T* src = static_cast<const T*>(a.q) + seq * a.q_row + head * a.q_head + D / 4 * (lane >> 4);
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
    if (live) r.x[j] = *reinterpret_cast<const typename Vec8<T>::type*>(src + 8 * j);
  return r;
}
template <class T, int D>
__device__ __forceinline__ float q4_queries(const Q4Attn& a, const Q4Query<T, D>& in, h8v (&q)[D / 32]) {
  float f[D / 32][8], big = 0.f;
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f[j][e] = a.scale < 0.f ? -static_cast<float>(in.x[j][e]) : static_cast<float>(in.x[j][e]);
      big = fmaxf(big, __builtin_fabsf(f[j][e]));
    }
  }
  float factor = __builtin_fabsf(a.scale);
  if constexpr (!__is_same(T, _Float16)) {
    big = xor_max<32>(xor_max<16>(big));
    const int ex = big < INFINITY ? __builtin_amdgcn_frexp_expf(big) : 0;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) f[j][e] = __builtin_amdgcn_ldexpf(f[j][e], -ex);
    factor = __builtin_amdgcn_ldexpf(factor, ex);
  }
  factor = fminf(fmaxf(factor * kLog2e, 1e-30f), __FLT_MAX__);
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      q[j][2 * e] = f2h(f[j][e]);
      q[j][2 * e + 1] = f2h(f[j][e + 4]);
    }
  return factor;
}

// Tiles first, first + step, ... below `end` of an item with `keys` keys; fresh: the row that is written now, or -1.
// Each half of a tile's registers is loaded again as soon as it is used up: K's while weights and values are worked
// on, V's while the next tile's scores are.
template <class T, int D>
__device__ __forceinline__ void q4_tiles(const Q4Attn& a, int seq, int kvh, int first, int step, int end, int keys, int fresh,
                                         const h8v (&q)[D / 32], float factor,
                                         int lane, Q4State<D>& st) {
#pragma unroll
  for (int h = 0; h < D / 64; ++h)
#pragma unroll
    for (int j = 0; j < 4; ++j) st.o[h][j] = f4v{0.f, 0.f, 0.f, 0.f};
  st.m = -INFINITY;
  st.l = 0.f;
  const int all = (keys + kTileKeys - 1) / kTileKeys, tiles = min(end, all);
  if (first >= tiles) return;
  const int64_t hr = (static_cast<int64_t>(seq) * a.c.heads + kvh) * a.c.max_len;
  const Q4Base b = q4_base<D>(a.c, hr, lane);
  Q4Tile<D> x;
  f4v s[2];
  q4_load_k<D>(b, first, x);
  q4_load_v<D>(b, first, x);
  int t = first;
  for (; t + step < tiles; t += step) {
    q4_scores<D>(x, q, s);
    q4_load_k<D>(b, t + step, x);
    q4_values<D, false>(x, s, factor, 0, lane, st);
    q4_load_v<D>(b, t + step, x);
  }
  const int left = keys - t * kTileKeys;
  if (fresh >= 0 && t == all - 1) q4_fresh<T, D>(a, q4_fresh_values<T, D>(a, seq, kvh, lane), hr, fresh, lane, x);
  q4_scores<D>(x, q, s);
  if (left >= kTileKeys) q4_values<D, false>(x, s, factor, 0, lane, st);
  else q4_values<D, true>(x, s, factor, left, lane, st);
}

// Where the waves' results of an item meet; `cols` query heads of it.
template <int D>
struct Q4Merge {
  static constexpr int kPitch = D + 4;  // 16 lanes' rows on different banks
  float *acc, *m, *l;                   // [waves][cols][kPitch], [waves][16], [waves][16]
  __device__ Q4Merge(float* lds, int waves, int cols) : acc(lds + 2 * waves * kCols), m(lds), l(lds + waves * kCols) {}
  static constexpr int bytes(int waves, int cols) { return 4 * waves * (2 * kCols + cols * kPitch); }
};

template <int D>
__device__ __forceinline__ void q4_hand_in(const Q4Merge<D>& x, const Q4State<D>& st, int wave, int cols, int lane) {
  const int h = lane & 15, g = lane >> 4;
  const float l = xor_add<32>(xor_add<16>(st.l));
  if (h >= cols) return;
  if (g == 0) {
    x.m[wave * kCols + h] = st.m;
    x.l[wave * kCols + h] = l;
  }
  float* to = x.acc + (wave * cols + h) * Q4Merge<D>::kPitch + 16 * g;
#pragma unroll
  for (int half = 0; half < D / 64; ++half)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<f4v*>(to + 64 * half + 4 * r) =
          f4v{st.o[half][0][r], st.o[half][1][r], st.o[half][2][r], st.o[half][3][r]};
}

// The sum over the waves for query head h and dim d: (m, l, o) with o, l relative to exp2(m).
template <int D>
__device__ __forceinline__ float q4_sum(const Q4Merge<D>& x, int waves, int cols, int h, int d, float& m, float& l) {
  m = -INFINITY;
  for (int w = 0; w < waves; ++w) m = fmaxf(m, x.m[w * kCols + h]);
  float o = 0.f;
  l = 0.f;
  for (int w = 0; w < waves; ++w) {
    const float mw = x.m[w * kCols + h], e = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - m);
    l = fmaf(e, x.l[w * kCols + h], l);
    o = fmaf(e, x.acc[(w * cols + h) * Q4Merge<D>::kPitch + d], o);
  }
  return o;
}

// An item's place: query heads [head, head + cols) of key/value head kvh.
struct Q4Item {
  int kvh, head, cols;
};
__device__ __forceinline__ int q4_cols(const Q4Attn& a) { return min(kCols, a.heads / a.c.heads); }  // of the largest item
__device__ __forceinline__ Q4Item q4_item(const Q4Attn& a, int item) {
  const int group = a.heads / a.c.heads, parts = (group + kCols - 1) / kCols;
  const int kvh = item / parts, first = item % parts * kCols;
  return Q4Item{kvh, kvh * group + first, min(kCols, group - first)};
}

template <class T>
__device__ __forceinline__ void q4_store(const Q4Attn& a, int seq, int head, int d, float o, float l) {
  static_cast<T*>(a.out)[seq * a.o_row + head * a.o_head + d] = static_cast<T>(l == 0.f ? 0.f : o / l);
}

// Inclusive sum over the wave by DPP: within rows of 16 lanes, then row 0 to 1 and 2 to 3, then the lower half to the
// upper. (Shuffles go through the LDS pipe: a microsecond in the 12000 blocks of 200 sequences.)
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);   // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);   // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);   // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 to rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 to rows 2 and 3
  return v;
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

// How the keys of all sequences are shared out: chunks so long that about kWantBlocks blocks have one (two a CU), at least
// two tiles a wave and at most a.chunk. Lane i has the keys of sequences i, i + 64, .. Many items fill the CUs in any
// case and get a.chunk, without the sum over the lengths, unless the cache is so long that it makes a.chunk long (q4_plan);
// more sequences than kLookThrough nobody looks through at all.
// (One sequence of 3000 keys in a cache for 131072, 8 heads of 128: 11.0 us, in chunks for a full cache 18.9; 8 of 2000
// for 32768 12.3 against 17.1; 32 ragged ones of up to 4000 16.3 against 19.5; lengths near the full ones are alike.)
constexpr int kLookThrough = 256, kRounds = kLookThrough / 64, kWantBlocks = 512;
struct Q4Share {
  int keys[kRounds], chunk;
};
__device__ __forceinline__ Q4Share q4_share(const Q4Attn& a, int items, int lane) {
  Q4Share x;
  x.chunk = a.chunk;
  if (a.c.n_seq > kLookThrough) return x;
  float all = 0.f;
#pragma unroll
  for (int j = 0; j < kRounds; ++j) {
    int fresh;
    x.keys[j] = 0;
    if (64 * j < a.c.n_seq && 64 * j + lane < a.c.n_seq) x.keys[j] = q4_keys(a, 64 * j + lane, fresh);
    all += static_cast<float>(x.keys[j]);
  }
  if (!a.unit) return x;
  const float want = fminf(group_sum<64>(all) * static_cast<float>(items) * (1.0f / kWantBlocks), static_cast<float>(a.chunk));
  x.chunk = min(max((static_cast<int>(want) / a.unit + 1) * a.unit, 2 * a.unit), a.chunk);
  return x;
}

// The piece of work of number `piece`: a sequence and the first key of its chunk; false where there is none. The full
// chunks of all sequences come first and are spread over the CUs while these are empty; then the rest of every
// sequence (or its zeros); blocks without work come last, behind everything.
__device__ __forceinline__ bool q4_piece(const Q4Attn& a, const Q4Share& x, int piece, int lane, int& seq, int& begin) {
  int fresh;
  if (a.c.n_seq > kLookThrough) {  // chunk by chunk
    seq = piece % a.c.n_seq;
    begin = piece / a.c.n_seq * x.chunk;
    return begin == 0 || begin < q4_keys(a, seq, fresh);
  }
  int full = 0;  // chunks of the sequences so far
#pragma unroll
  for (int j = 0; j < kRounds; ++j) {
    if (64 * j >= a.c.n_seq) break;
    const int n = x.keys[j] / x.chunk, incl = wave_scan(n) + full;
    const uint64_t past = __builtin_amdgcn_ballot_w64(incl > piece);
    if (past) {
      const int at = __builtin_ctzll(past);
      seq = 64 * j + at;
      begin = (piece - (__builtin_amdgcn_readlane(incl, at) - __builtin_amdgcn_readlane(n, at))) * x.chunk;
      return true;
    }
    full = __builtin_amdgcn_readlane(incl, 63);
  }
  seq = piece - full;
  if (seq >= a.c.n_seq) return false;
  const int keys = q4_keys(a, seq, fresh), rest = keys % x.chunk;
  begin = keys - rest;
  return rest > 0 || keys == 0;
}

// Where the chunks of a sequence are in the workspace: by their pieces' numbers, or, where all chunks have one size, by
// sequence, so that nobody needs the other lengths.
struct Q4Chunks {
  int n, full, first, last;
  __device__ int at(int i) const { return i < full ? first + i : last; }
};
__device__ __forceinline__ Q4Chunks q4_chunks(const Q4Attn& a, int items, int seq, int lane) {
  int fresh;
  const int keys = q4_keys(a, seq, fresh);
  if (!a.unit) {
    const int n = keys / a.chunk + (keys % a.chunk != 0);
    return Q4Chunks{n, n, seq * a.most, 0};
  }
  const Q4Share x = q4_share(a, items, lane);
  int before = 0, all = 0;
#pragma unroll
  for (int j = 0; j < kRounds; ++j) {
    if (64 * j >= a.c.n_seq) break;
    const int here = x.keys[j] / x.chunk;
    before += 64 * j + lane < seq ? here : 0;
    all += here;
  }
  const int full = keys / x.chunk;
  return Q4Chunks{full + (keys % x.chunk != 0), full, wave_total(before), wave_total(all) + seq};
}

// The first arguments, which arrive in scalar registers, are what the way to the first tile needs; the rest of `a`
// is read from memory meanwhile.
template <class T, int D>
__global__ void __launch_bounds__(512, 4) q4_attention_kernel(const int64_t* lens, uint8_t* k_codes, _Float16* k_meta,
                                                              uint8_t* v_codes, _Float16* v_meta, int max_len, int kv_heads,
                                                              int heads, int pieces, int items, Q4Attn a) {
  extern __shared__ float lds[];
  a.lens = lens;
  a.c.k_codes = k_codes;
  a.c.k_meta = k_meta;
  a.c.v_codes = v_codes;
  a.c.v_meta = v_meta;
  a.c.max_len = max_len;
  a.c.heads = kv_heads;
  a.heads = heads;
  a.pieces = pieces;
  const int waves = blockDim.x / 64, item = blockIdx.x % items, piece = blockIdx.x / items;
  const int lane = threadIdx.x & 63;
  int seq = piece, begin = 0, chunk = max_len;
  if (pieces) {
    const Q4Share share = q4_share(a, items, lane);
    if (!q4_piece(a, share, piece, lane, seq, begin)) return;
    chunk = share.chunk;
  }
  const Q4Item it = q4_item(a, item);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int fresh;
  // requested before the length is known
  const Q4Query<T, D> query = q4_load_query<T, D>(a, seq, it.head + (lane & 15), (lane & 15) < it.cols, lane);
  const int keys = q4_keys(a, seq, fresh);
  h8v q[D / 32];
  const float factor = q4_queries<T, D>(a, query, q);
  Q4State<D> st;
  q4_tiles<T, D>(a, seq, it.kvh, begin / kTileKeys + wave, waves, (begin + chunk) / kTileKeys, keys, fresh, q, factor, lane,
                 st);
  const Q4Merge<D> x(lds, waves, it.cols);
  q4_hand_in<D>(x, st, wave, it.cols, lane);
  __syncthreads();
  const bool whole = keys <= chunk;
  const int64_t slot = static_cast<int64_t>(a.unit ? piece : seq * a.most + begin / chunk) * items + item;
  const int cols = q4_cols(a);
  float* ml = a.ws + static_cast<int64_t>(pieces) * items * cols * D + slot * cols * 2;
  for (int i = threadIdx.x; i < it.cols * D; i += blockDim.x) {
    float m, l;
    const int h = i / D, d = i % D;
    const float o = q4_sum<D>(x, waves, it.cols, h, d, m, l);
    if (whole) {
      q4_store<T>(a, seq, it.head + h, d, o, l);
    } else {
      a.ws[slot * cols * D + i] = o;
      if (d == 0) {
        ml[2 * h] = m;
        ml[2 * h + 1] = l;
      }
    }
  }
}

// Joins the chunks of items that have several: block = (query head, sequence). The chunks' O are requested before
// their weights are known. (A block for all query heads of an item is slower, its heads waiting for each other:
// 7.7 us against 5.0 for 64 ragged sequences of 32 heads.)
// 512 threads where the blocks are at most one a CU, so that twice the chunks are on their way (2 sequences of 39000 keys,
// one key/value head: the call takes 14.8 us instead of 18.4; 1024 threads 14.2, but 10.3 instead of 9.6 where
// there are fewer chunks), else 256 (64 ragged sequences of 32 heads 28.5 against 30.2).
constexpr int kBatch = 8;
template <class T, int D, int kCombine>
__global__ void __launch_bounds__(kCombine) q4_combine_kernel(const int64_t* lens, Q4Attn a) {
  constexpr int kLanes = kCombine / D;
  __shared__ float red[2][kCombine / 64], part[kLanes][D];
  extern __shared__ float weight[];  // [the most chunks of a sequence]
  const int seq = blockIdx.y, head = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid / 64, d = tid % D, from = tid / D;
  a.lens = lens;
  const int group = a.heads / a.c.heads, parts = (group + kCols - 1) / kCols, items = a.c.heads * parts, cols = q4_cols(a);
  const Q4Chunks at = q4_chunks(a, items, seq, lane);
  const int n = at.n;
  if (n <= 1) return;  // its block finished it
  const int in_group = head % group, item = head / group * parts + in_group / kCols, h = in_group % kCols;
  const float2* ml = reinterpret_cast<const float2*>(a.ws + static_cast<int64_t>(a.pieces) * items * cols * D) + item * cols + h;
  const float* acc = a.ws + static_cast<int64_t>(item * cols + h) * D + d;
  const auto slot = [&](int i) { return static_cast<int64_t>(at.at(i)) * (items * cols); };
  const auto load = [&](int i, float (&x)[kBatch]) {  // chunks i, i + kLanes, ..; past the end the last one
#pragma unroll
    for (int j = 0; j < kBatch; ++j) x[j] = acc[slot(min(i + j * kLanes, n - 1)) * D];
  };
  float x[kBatch];
  load(from, x);
  float m = -INFINITY, l = 0.f;
  for (int i = tid; i < n; i += kCombine) {
    weight[i] = ml[slot(i)].x;
    m = fmaxf(m, weight[i]);
  }
  m = group_max<64>(m);
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kCombine / 64; ++i) m = fmaxf(m, red[0][i]);
  for (int i = tid; i < n; i += kCombine) {
    weight[i] = __builtin_amdgcn_exp2f(weight[i] - m);
    l = fmaf(weight[i], ml[slot(i)].y, l);
  }
  l = group_sum<64>(l);
  if (lane == 0) red[1][wave] = l;
  __syncthreads();
  float o = 0.f;
  for (int i = from;;) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (i + j * kLanes < n) o = fmaf(weight[i + j * kLanes], x[j], o);
    i += kBatch * kLanes;
    if (i >= n) break;
    load(i, x);
  }
  part[from][d] = o;
  __syncthreads();
  if (tid >= D) return;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < kCombine / 64; ++i) l += red[1][i];
#pragma unroll
  for (int j = 1; j < kLanes; ++j) o += part[j][d];
  q4_store<T>(a, seq, head, d, o, l);
}

// What of a call goes by sizes alone (the lengths are on the device). A cache of up to kOneChunk rows is one
// chunk: a second launch to join chunks costs more than it gains there (16 sequences x 20 heads of 64 over 1500 keys
// 13.6 us in one chunk, 18.9 shared out further; 1 x 20 8.4 and 9.3). For heads of 128, which take a wave twice as long, half
// of that where the items fill a quarter of the CUs at most (2000 keys x 8 heads: 9.5 us, in one chunk 13.2; 32 x 8 heads over
// 1536 keys 20.1, in one 13.4). Longer ones are cut. The largest chunk gives full lengths about
// kWantBlocks blocks (131000 keys x 8 heads of 128: 42.8 us, with twice the blocks 51.7), but has at most kWaveKeys or
// kManyWaveKeys keys a wave, which bounds how long a few long sequences among short ones keep their CUs (64 ragged
// sequences of up to 8000 keys x 8 heads of 128 with 128 / 192 / 256 keys a wave: 29.4 / 28.6 / 30.6 us, 64 of 8000: 134.7 /
// 131.9 / 129.9). The chunk is at least 1 / kMostBlocks of everything, which bounds the workspace and comes before that; where
// this makes it kLoose times as long as the bound for many items, up to kLookThrough sequences get chunks by their lengths (64
// ragged sequences x 8 heads of 128 in caches of 16384 / 32768 / 49152 / 131072 rows, 1.3 / 2.7 / 4 / 11 times the bound: 25.5 /
// 32.0 / 31.2 / 53.2 us, by length 26.3 / 26.9 / 26.5 / 26.8; all of 1000 keys 22.1 / 23.5 / 22.4 / 28.7 and 24.8 / 25.9 / 25.1 /
// 26.6; 250 x 4 heads, one of 8000 keys, 2.6 / 5.2 / 10 times: 25.0 / 29.6 / 49.7, by length 28.5 / 28.7 / 28.7). Blocks
// have 8 waves where items are few and 4 where they fill the CUs anyway (those 64 ragged sequences: 33.5 us against 39.5; 64 x 20 heads of 64 over
// 700 keys 15.0 against 17.2, but 16 x 20 over 1500 keys as two chunks of 4 waves 16.3 against 13.6), or where the merge of
// 16 heads of 128 would pass 64 KB of LDS.
struct Q4Plan {
  int items, cols, waves, chunk, most, unit, pieces;
  int64_t blocks(int n_seq) const { return static_cast<int64_t>(items) * (pieces ? pieces : n_seq); }
};
constexpr int kOneChunk = 2048, kWaveKeys = 256, kManyWaveKeys = 192, kMostBlocks = 8192, kManyItems = 512, kLoose = 3;

Q4Plan q4_plan(int n_seq, int heads, int kv_heads, int max_len, int dim) {
  Q4Plan p;
  const int group = heads / kv_heads;
  p.items = kv_heads * ((group + kCols - 1) / kCols);
  p.cols = min(kCols, group);
  const int lds8 = dim == 64 ? Q4Merge<64>::bytes(8, p.cols) : Q4Merge<128>::bytes(8, p.cols);
  const bool many = static_cast<int64_t>(n_seq) * p.items >= kManyItems;
  p.waves = min(max_len / kTileKeys, many || lds8 > 65536 ? 4 : 8);
  p.chunk = max_len;
  p.most = 1;
  p.unit = p.pieces = 0;
  const bool few_items = static_cast<int64_t>(n_seq) * p.items <= 64;
  if (max_len <= (dim == 128 && few_items ? kOneChunk / 2 : kOneChunk)) return p;
  const int64_t keys = static_cast<int64_t>(n_seq) * p.items * max_len, unit = kTileKeys * p.waves;
  const int64_t most = (many ? kManyWaveKeys : kWaveKeys) * p.waves;  // (std:: below: the unqualified ones take ints on the host)
  const int64_t want = std::min<int64_t>(std::max(std::min(keys / kWantBlocks, most), keys / kMostBlocks), max_len);
  p.chunk = static_cast<int>((want + unit) / unit * unit);
  // full chunks: of the largest n_seq max_len / chunk, of smaller ones no more than kWantBlocks / items (none of more
  // items than that: a chunk is then longer than all sequences); a rest each
  const int full = max_len / p.chunk, few = p.items > kWantBlocks ? 0 : kWantBlocks / p.items + 1;
  const bool by_length = n_seq <= kLookThrough && (!many || want > kLoose * most);
  p.most = (by_length ? max(full, few) : full) + 1;
  if (by_length) p.unit = static_cast<int>(unit);
  const int64_t all_full = static_cast<int64_t>(n_seq) * full;
  const int64_t pieces = n_seq + (by_length ? std::max<int64_t>(all_full, few) : all_full);
  p.pieces = static_cast<int>(std::min<int64_t>(pieces, 0x7FFFFFFF));
  return p;
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

constexpr int kMaxLen = 1 << 30;  // a row and a chunk further fit 32 bits

// What every entry point asks of a cache; FW_OK or FW_EINVAL.
int check_cache(const char* what, const Q4Cache& c, int dim) {
  if (!c.k_codes || !c.k_meta || !c.v_codes || !c.v_meta) return fw_fail(FW_EINVAL, "%s: null cache pointer", what);
  if (c.n_seq <= 0 || c.heads <= 0) return fw_fail(FW_EINVAL, "%s: n_seq and kv_heads must be positive", what);
  if (dim != 64 && dim != 128) return fw_fail(FW_EINVAL, "%s: head_dim must be 64 or 128", what);
  if (c.max_len <= 0 || c.max_len % 32 || c.max_len > kMaxLen)
    return fw_fail(FW_EINVAL, "%s: max_len must be a positive multiple of 32 up to 2^30", what);
  if (!aligned(c.k_codes, 16) || !aligned(c.k_meta, 16) || !aligned(c.v_codes, 16) || !aligned(c.v_meta, 16))
    return fw_fail(FW_EINVAL, "%s: the cache must be 16-byte aligned", what);
  return FW_OK;
}

// Rows whose 8-element pieces are 16-byte accesses.
bool rows_ok(const void* p, int64_t row, int64_t head) { return aligned(p, 16) && row % 8 == 0 && head % 8 == 0; }

// launch(T(), integral_constant D) for a dtype and a head size.
template <class F>
void q4_by_type(int dtype, int dim, F launch) {
  const std::integral_constant<int, 64> d64;
  const std::integral_constant<int, 128> d128;
  if (dtype == FW_F16 && dim == 64) launch(_Float16(), d64);
  else if (dtype == FW_F16) launch(_Float16(), d128);
  else if (dim == 64) launch(__bf16(), d64);
  else launch(__bf16(), d128);
}

// Waves of the append and the read: one each for every (head, half) of a slot, or for the read kParts of them where
// that would be more than 32 a CU, so that a wave has more loads on their way behind its search for the sequence
// (8 x 1500 rows of 20 heads of 64: 13.6 us against 15.4; the append, 19.4 and 19.9, has most of its time after
// the loads, and 96 K rows of 8 heads of 128 take it 31.9 and 29.8).
constexpr int kParts = 2, kFewUnits = 8192;
struct Q4Grid {
  int64_t slots;
  int parts;
  unsigned blocks;
};
Q4Grid q4_grid(int64_t rows, int n_seq, int heads, int dim, int most_parts) {
  Q4Grid g;
  const int per_slot = heads * (dim / 64);
  g.slots = rows / 8 + 2 * static_cast<int64_t>(n_seq);
  g.parts = g.slots * per_slot > kFewUnits ? most_parts : 1;
  g.blocks = static_cast<unsigned>((g.slots * ((per_slot + g.parts - 1) / g.parts) + 3) / 4);
  return g;
}

int check_packed(const char* what, const Q4Rows& r, const int64_t* cu, const int64_t* pos, int64_t rows, const Q4Cache& c,
                 int dim, int dtype) {
  if (const int rc = check_cache(what, c, dim)) return rc;
  if (dtype != FW_F16 && dtype != FW_BF16) return fw_fail(FW_EINVAL, "%s: dtype must be FW_F16 or FW_BF16", what);
  if (rows < 0) return fw_fail(FW_EINVAL, "%s: rows must not be negative", what);
  if (!cu || !pos || (rows > 0 && (!r.k || !r.v))) return fw_fail(FW_EINVAL, "%s: null pointer", what);
  if (rows > 0 && (!rows_ok(r.k, r.k_row, r.k_head) || !rows_ok(r.v, r.v_row, r.v_head)))
    return fw_fail(FW_EINVAL, "%s: k and v must be 16-byte aligned with strides in multiples of 8", what);
  // the grid: 4 waves a block, slots x heads x halves waves (a quotient: their product may pass 64 bits)
  const int64_t slots = rows / 8 + 2 * static_cast<int64_t>(c.n_seq), per_slot = static_cast<int64_t>(c.heads) * (dim / 64);
  if (slots > 0xFFFFFFFFll / 256 * 4 / per_slot)
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
  const Q4Grid g = q4_grid(rows, n_seq, kv_heads, head_dim, 1);
  q4_by_type(dtype, head_dim, [&](auto t, auto d) {
    hipLaunchKernelGGL((kv_q4_append_kernel<decltype(t), d.value>), dim3(g.blocks), dim3(256), 0, stream, cu, pos, rows, g.slots,
                       n_seq, kv_heads, r, c);
  });
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
  const Q4Grid g = q4_grid(rows, n_seq, kv_heads, head_dim, kParts);
  q4_by_type(dtype, head_dim, [&](auto t, auto d) {
    const auto kernel = g.parts == 1 ? kv_q4_read_kernel<decltype(t), d.value, 1> : kv_q4_read_kernel<decltype(t), d.value, kParts>;
    hipLaunchKernelGGL(kernel, dim3(g.blocks), dim3(256), 0, stream, cu, pos, rows, g.slots, n_seq, kv_heads, r, c);
  });
  return fw_check_launch("kv_q4_read");
}

extern "C" int64_t fw_decode_attention_q4_ws_floats(int n_seq, int heads, int kv_heads, int max_len, int head_dim) {
  if (n_seq <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || max_len <= 0 || max_len % 32 ||
      max_len > kMaxLen || (head_dim != 64 && head_dim != 128))
    return 0;
  const Q4Plan p = q4_plan(n_seq, heads, kv_heads, max_len, head_dim);
  return p.pieces ? (p.blocks(n_seq) * p.cols * (head_dim + 2) + 3) / 4 * 4 : 4;
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
  if (!(__builtin_fabsf(scale) < INFINITY)) return fw_fail(FW_EINVAL, "decode_attention_q4: scale must be finite");
  if (!k_new != !v_new) return fw_fail(FW_EINVAL, "decode_attention_q4: k_new and v_new must be given together");
  if (heads <= 0 || heads % kv_heads) return fw_fail(FW_EINVAL, "decode_attention_q4: heads must be a multiple of kv_heads");
  if (!rows_ok(q, q_row, q_head) || !rows_ok(out, o_row, o_head) ||
      (k_new && (!rows_ok(k_new, k_row, k_head) || !rows_ok(v_new, v_row, v_head))))
    return fw_fail(FW_EINVAL,
                   "decode_attention_q4: q, out, k_new and v_new must be 16-byte aligned with strides in multiples of 8");
  const int64_t need = fw_decode_attention_q4_ws_floats(n_seq, heads, kv_heads, max_len, head_dim);
  if (!ws || ws_floats < need || !aligned(ws, 16))
    return fw_fail(FW_EINVAL, "decode_attention_q4: workspace needs %lld floats, 16-byte aligned", static_cast<long long>(need));
  const Q4Plan p = q4_plan(n_seq, heads, kv_heads, max_len, head_dim);
  if (n_seq > 65535 || !grid_ok(p.blocks(n_seq), 64 * p.waves))
    return fw_fail(FW_EINVAL, "decode_attention_q4: too many sequences");
  const int threads = heads * static_cast<int64_t>(n_seq) <= 256 ? 512 : 256;  // of the combine launch
  if (p.pieces && !grid_ok(heads, threads)) return fw_fail(FW_EINVAL, "decode_attention_q4: too many heads");
  const Q4Attn a{q, out, q_row, q_head, o_row, o_head, Q4Rows{k_new, v_new, k_row, k_head, v_row, v_head}, lens, c, heads, scale,
                 p.chunk, p.most, p.unit, p.pieces, ws};
  const int lds = head_dim == 64 ? Q4Merge<64>::bytes(p.waves, p.cols) : Q4Merge<128>::bytes(p.waves, p.cols);
  q4_by_type(dtype, head_dim, [&](auto t, auto d) {
    hipLaunchKernelGGL((q4_attention_kernel<decltype(t), d.value>), dim3(static_cast<unsigned>(p.blocks(n_seq))),
                       dim3(64 * p.waves), lds, stream, lens, c.k_codes, c.k_meta, c.v_codes, c.v_meta, max_len, kv_heads, heads, p.pieces, p.items, a);
  });
  if (const int rc = fw_check_launch("decode_attention_q4")) return rc;
  if (!p.pieces) return FW_OK;
  q4_by_type(dtype, head_dim, [&](auto t, auto d) {
    const auto kernel = threads == 512 ? q4_combine_kernel<decltype(t), d.value, 512> : q4_combine_kernel<decltype(t), d.value, 256>;
    hipLaunchKernelGGL(kernel, dim3(heads, n_seq), dim3(threads), 4 * p.most, stream, lens, a);
  });
  return fw_check_launch("decode_attention_q4 combine");
}
