// Single-token attention over a key/value cache in pages (pages.h) for gfx950, the rows that a group of sequences shares
// read once for all of it. Built with MFMA results in VGPRs, as the other attentions.
#include <algorithm>
#include <type_traits>

#include "lds_pipe.h"
#include "packed_rows.h"
#include "pages.h"

namespace fw {
namespace {

typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));

template <class T>
struct Types;
template <>
struct Types<_Float16> {
  typedef h8v v8;
  typedef h2v v2;
  static constexpr float kSlack = 3.f, kLift = 8.f;
};
template <>
struct Types<__bf16> {
  typedef b8v v8;
  typedef b2v v2;
  static constexpr float kSlack = 8.f, kLift = 0.f;
};

__device__ __forceinline__ f4v mfma16(const h8v& a, const h8v& b, const f4v& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f4v mfma16(const b8v& a, const b8v& b, const f4v& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float add_pair(h2v x, float s) {
  return __builtin_amdgcn_fdot2(x, h2v{static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)}, s, false);
}
__device__ __forceinline__ float add_pair(b2v x, float s) {
  return __builtin_amdgcn_fdot2_f32_bf16(x, b2v{static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)}, s, false);
}

// ------------------------------------------------------------------------------------------
// A piece of work is a run of keys of one sequence's table and the columns that see them: a column is a query head of a
// sequence, and the `group` heads that share a key/value head, of the sequence alone or of all sequences of its group one after
// another, are the columns of the products S^T = K Q^T and O^T = V^T P^T (16 keys or head dims by 16 columns). A wave takes
// 32 keys at a time, straight from the pages into the operands' registers:
//  - K: row i of the first 16 is key 8 (i / 4) + i % 4, of the second 4 more, so that lane group g = lane / 16 ends with the
//    scores of keys 8 g .. 8 g + 7 for column lane % 16: what the P V products take from it, without crossing lanes.
//  - V: a lane's 8 keys of a dim are 16 bytes of a page.
//  - Weights are exp2(score - m), m the running maximum less kLift (log2 units), which only moves when a score passes the maximum
//    by kSlack; they are rounded to the type, which the matrix instructions take, and their sum, in fp32, is over the rounded
//    ones. fp16 ones, lifted by 2^8, keep all bits of the type from 2^-22 of the maximum on, and smaller ones are multiples of 2^-32
//    of it (without it that begins at 2^-14, and many keys far below one lose or gain half their sum). They stay in the type as
//    long as scores are defined: below 2^27 in size m, rounded to fp32, is off by at most 4, and moves once a score passes it by 4
//    (3 as it is rounded there; above 2^26 at once), so the largest exponent is 14 (with a slack of 8 20, past the type).
// Bound by memory where there is much to read (17 sequences of up to 48000 rows in groups of 1 to 7, 64 query heads over 8 of 128:
// 409 MB in 88 us, 4.6 TB/s, with the joining; 16 of 1500 rows x 20 heads of 64 28 us, 4.4 TB/s), else by the chain of dependent
// loads (lengths, table, keys, results of the pieces), about 10 us in two launches, 5 in one.
// ------------------------------------------------------------------------------------------
struct PagedArgs {
  const void *q, *k, *v;
  void* out;
  int64_t q_row, q_head, o_row, o_head;
  const int32_t* table;
  const int64_t *lens, *cu_g, *shared;
  int n_seq, heads, kv_heads, groups, width, n_pages, page_shift;
  float scale;
  int cols;           // columns of a piece of a group's shared keys, at most: 16, or 64 or 128 in wide ones
  int want;           // pieces that all keys are to make, about
  uint32_t unit;      // what a chunk of keys is a multiple of: a tile for each wave
  int most;           // pieces there may be; 0: each sequence is a piece, and nothing is shared
  int* plan;          // the number of Pieces, they from word 4 on, Owners, and the plan's arrays where LDS does not hold them
  float *part, *ml;   // O [slot][kv head][16][D], (m, l) [slot][kv head][16][2]
};

constexpr int kTileKeys = 32;
constexpr int kCols = 16;
constexpr float kLog2e = 1.4426950408889634f;

// Columns [col, col + cols) of the sequences from `seq` on see keys [begin, end) of the table of sequence `table`, the first of them
// that is not idle.
struct __align__(16) Piece {
  int seq, col, cols, begin;
  int end, slot;  // where 16 columns' results go, cols / 16 slots; -1: they are the whole, and go to `out`
  int table, pad;
};
// What the pieces of a sequence left: of its group's shared keys, its columns from `col` on in runs of `step` slots, and its own.
struct __align__(16) Owner {
  int shared_slot, shared_n, shared_step, col;
  int slot, n;
  int pad[2];
};

// The keys that a sequence sees, 0 for an idle one.
__device__ __forceinline__ int paged_keys(const PagedArgs& a, int seq) {
  return static_cast<int>(within(a.lens[seq], 0, static_cast<int64_t>(a.width) << a.page_shift));
}

template <class T, int D, int CT>
struct PagedState {
  f4v o[CT][D / 16];  // lane (column, g), register r: dim 16 db + 4 g + r
  float m[CT], l[CT];  // l: this lane's keys only
};

template <class T, int D>
struct PagedTile {
  typename Types<T>::v8 k[2][D / 32], v[D / 16];
};

// Where the pages of a wave's next 64 tiles are, lane l its l-th; a page of 16 rows is half a tile. -1: no page.
struct PagedPages {
  int lo, hi;
};
__device__ __forceinline__ PagedPages paged_pages(const PagedArgs& a, const int32_t* table, int tile, int end) {
  const int row = tile * kTileKeys;
  PagedPages p{-1, -1};
  if (row >= 0 && row < end) p.lo = table[row >> a.page_shift];
  if (a.page_shift == 4 && row >= 0 && row + 16 < end) p.hi = table[(row >> 4) + 1];
  if (a.page_shift != 4) p.hi = p.lo;
  if (p.lo < 0 || p.lo >= a.n_pages) p.lo = -1;
  if (p.hi < 0 || p.hi >= a.n_pages) p.hi = -1;
  return p;
}

// A tile whose rows lie in pages lo and hi (no page: page 0 is read, and none of it counts): the lane's two rows of K, its unit of V.
template <class T, int D>
__device__ __forceinline__ void paged_load_k(const PagedArgs& a, int kvh, int tile, int lo, int hi, int lane, PagedTile<T, D>& t) {
  typedef typename Types<T>::v8 v8;
  const int i = lane & 15, g = lane >> 4, page = i < 8 ? lo : hi, rows = 1 << a.page_shift;
  const int row = (tile * kTileKeys + 8 * (i >> 2) + (i & 3)) & (rows - 1);
  const T* at = static_cast<const T*>(a.k) + ((static_cast<int64_t>(max(page, 0)) * a.kv_heads + kvh) * rows + row) * D + 8 * g;
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int j = 0; j < D / 32; ++j) t.k[s][j] = *reinterpret_cast<const v8*>(at + 4 * s * D + 32 * j);
}
template <class T, int D>
__device__ __forceinline__ void paged_load_v(const PagedArgs& a, int kvh, int tile, int lo, int hi, int lane, PagedTile<T, D>& t) {
  typedef typename Types<T>::v8 v8;
  const int i = lane & 15, g = lane >> 4, page = g < 2 ? lo : hi, rows = 1 << a.page_shift;
  const int row = (tile * kTileKeys + 8 * g) & (rows - 1);
  const T* at = static_cast<const T*>(a.v) + ((static_cast<int64_t>(max(page, 0)) * a.kv_heads + kvh) * rows + row) * D + 8 * i;
#pragma unroll
  for (int db = 0; db < D / 16; ++db) t.v[db] = *reinterpret_cast<const v8*>(at + 128 * db);
}

// A tile's scores for the columns.
template <class T, int D, int CT>
__device__ __forceinline__ void paged_scores(const PagedTile<T, D>& t, const typename Types<T>::v8 (&q)[CT][D / 32], f4v (&s)[CT][2]) {
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) s[c][kt] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) s[c][kt] = mfma16(t.k[kt][j], q[c][j], s[c][kt]);
}

// Their weights and the sum over the values; MASKED: only the first `left` of the lane's 8 keys count.
template <class T, int D, int CT, bool MASKED>
__device__ __forceinline__ void paged_values(PagedTile<T, D>& t, f4v (&s)[CT][2], float factor, int left, PagedState<T, D, CT>& st) {
  typedef typename Types<T>::v8 v8;
  typedef typename Types<T>::v2 v2;
  v8 p[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    float top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (MASKED && 4 * kt + r >= left) s[c][kt][r] = -INFINITY;
        top = __builtin_elementwise_maximum(top, s[c][kt][r]);  // a NaN stays: its column is NaN anyway
      }
    top = fmaf(xor_max<32>(xor_max<16>(top)), factor, -Types<T>::kLift);
    if (__builtin_amdgcn_ballot_w64(top > st.m[c] + Types<T>::kSlack)) {
      const float m_new = fmaxf(st.m[c], top), corr = st.m[c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m[c] - m_new);
      st.l[c] *= corr;
#pragma unroll
      for (int db = 0; db < D / 16; ++db) st.o[c][db] *= corr;
      st.m[c] = m_new;
    }
    const float m = st.m[c] == -INFINITY ? 0.f : st.m[c];  // no key seen yet: the weights are 0
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        v2 x;
        x[0] = static_cast<T>(__builtin_amdgcn_exp2f(fmaf(s[c][kt][r], factor, -m)));
        x[1] = static_cast<T>(__builtin_amdgcn_exp2f(fmaf(s[c][kt][r + 1], factor, -m)));
        st.l[c] = add_pair(x, st.l[c]);
        p[c][4 * kt + r] = x[0];
        p[c][4 * kt + r + 1] = x[1];
      }
  }
#pragma unroll
  for (int db = 0; db < D / 16; ++db) {
    if constexpr (MASKED) {  // whatever the hidden rows hold, their values count as zeros
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e >= left) t.v[db][e] = static_cast<T>(0.f);
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) st.o[c][db] = mfma16(t.v[db], p[c], st.o[c][db]);
  }
}

// Tiles first, first + step, .. of the keys below `end` of a table. Each half of a tile's registers is loaded again as
// soon as it is used up.
template <class T, int D, int CT>
__device__ __forceinline__ void paged_tiles(const PagedArgs& a, const int32_t* table, int kvh, int first, int step, int end,
                                            const typename Types<T>::v8 (&q)[CT][D / 32], float factor, int lane,
                                            PagedState<T, D, CT>& st) {
#pragma unroll
  for (int c = 0; c < CT; ++c) {
#pragma unroll
    for (int db = 0; db < D / 16; ++db) st.o[c][db] = f4v{0.f, 0.f, 0.f, 0.f};
    st.m[c] = -INFINITY;
    st.l[c] = 0.f;
  }
  const int tiles = (end + kTileKeys - 1) / kTileKeys;
  if (first >= tiles) return;
  PagedPages pages = paged_pages(a, table, first + lane * step, end);
  int lo = __builtin_amdgcn_readlane(pages.lo, 0), hi = __builtin_amdgcn_readlane(pages.hi, 0);
  PagedTile<T, D> x;
  f4v s[CT][2];
  paged_load_k<T, D>(a, kvh, first, lo, hi, lane, x);
  paged_load_v<T, D>(a, kvh, first, lo, hi, lane, x);
  int t = first, n = 1;
  for (; t + step < tiles; t += step, ++n) {
    if ((n & 63) == 0) pages = paged_pages(a, table, t + step + lane * step, end);
    const int lo1 = __builtin_amdgcn_readlane(pages.lo, n & 63), hi1 = __builtin_amdgcn_readlane(pages.hi, n & 63);
    paged_scores<T, D, CT>(x, q, s);
    paged_load_k<T, D>(a, kvh, t + step, lo1, hi1, lane, x);
    if ((lo | hi) >= 0) paged_values<T, D, CT, false>(x, s, factor, 8, st);
    else paged_values<T, D, CT, true>(x, s, factor, (lane < 32 ? lo : hi) >= 0 ? 8 : 0, st);
    paged_load_v<T, D>(a, kvh, t + step, lo1, hi1, lane, x);
    lo = lo1;
    hi = hi1;
  }
  paged_scores<T, D, CT>(x, q, s);
  const int left = end - t * kTileKeys;
  if (left >= kTileKeys && (lo | hi) >= 0) paged_values<T, D, CT, false>(x, s, factor, 8, st);
  else paged_values<T, D, CT, true>(x, s, factor, (lane < 32 ? lo : hi) >= 0 ? left - 8 * (lane >> 4) : 0, st);
}

// The waves' results of 16 columns meet in LDS: O [wave][column][D + 4], m and l [wave][column].
template <int D>
struct PagedMerge {
  static constexpr int kPitch = D + 4;
  float *m, *l, *acc;
  int cols;
  __device__ PagedMerge(float* lds, int waves, int c) : m(lds), l(lds + waves * kCols), acc(lds + 2 * waves * kCols), cols(c) {}
  static constexpr int bytes(int waves, int cols) { return 4 * waves * (2 * kCols + cols * kPitch); }
};

__device__ __forceinline__ Piece* pieces_of(const PagedArgs& a) { return reinterpret_cast<Piece*>(a.plan + 4); }
__device__ __forceinline__ Owner* owners_of(const PagedArgs& a) { return reinterpret_cast<Owner*>(pieces_of(a) + a.most); }

// ------------------------------------------------------------------------------------------
// The plan turns the lengths into pieces. A group's shared rows are those that all its live sequences have, cut to whole
// tiles unless they are all that any of them has. All keys, times the runs of columns that see them, make about `want` pieces, a
// multiple of a tile for each wave; the pieces of one run of keys are alike, those of groups come first. Bound by latency, and a
// launch of its own costs as much as a small call's attention (6 to 8 us; a wave's own plan 2): up to 64 sequences and groups every
// wave of the attention makes the plan for itself, a sequence a lane, without barriers, and finds its block's piece in it
// (WavePlan); more of them are planned by one block, which leaves it in the workspace.
// ------------------------------------------------------------------------------------------
constexpr int kPlanThreads = 1024, kPlanLds = 1024;

// Words of its arrays: keys, groups of n sequences; starts, rows, low, high, live of the groups; the first piece of each.
__host__ __device__ constexpr int64_t plan_words(int64_t n, int64_t groups) { return 2 * n + 5 * groups + 1 + (n + groups + 1); }

struct Plan {
  const PagedArgs& a;
  int *keys, *of, *starts, *rows, *low, *high, *live, *before;  // low: the fewest keys, in the end whether no sequence sees more
  int groups, group, parts, total;
  uint32_t chunk;

  __device__ static int count(int x, uint32_t each) { return static_cast<int>((x + each - 1) / each); }
  __device__ int runs_of(int g) const { return ((starts[g + 1] - starts[g]) * group + a.cols - 1) / a.cols; }
  __device__ int begin_of(int s) const { return of[s] < 0 ? 0 : rows[of[s]]; }  // the sequence's first own row
  // where 16 columns' results of a piece go: one of a group has cols / 16 slots, one of a sequence one
  __device__ int slot_of(int at) const {
    const int shared = before[groups];
    return at < shared ? at * (a.cols / kCols) : shared * (a.cols / kCols) + (at - shared);
  }
  __device__ static int size_of(int keys, int n) { return ((keys + n - 1) / n + kTileKeys - 1) / kTileKeys * kTileKeys; }
  // What atomics made, read where they left it, which may be memory.
  __device__ static int made(const int* at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
  __device__ Piece piece(int at) const {
    const int e = find(before, groups + a.n_seq, at), s = e - groups, x = at - before[e];
    if (s < 0) {
      const int n = count(rows[e], chunk), runs = runs_of(e), i = x / runs, r = x % runs, size = size_of(rows[e], n);
      return Piece{starts[e], r * a.cols, min(a.cols, (starts[e + 1] - starts[e]) * group - r * a.cols), i * size,
                   min((i + 1) * size, rows[e]), low[e] && n == 1 ? -1 : slot_of(at), made(live + e), 0};
    }
    const int n = (before[e + 1] - before[e]) / parts, begin = begin_of(s), mine = max(keys[s] - begin, 0), i = x / parts, r = x % parts;
    const int size = size_of(mine, n);
    return Piece{s, r * kCols, min(kCols, group - r * kCols), begin + i * size, begin + min((i + 1) * size, mine),
                 begin == 0 && n == 1 ? -1 : slot_of(at), s, 0};
  }
  __device__ Owner owner(int s) const {
    Owner o{};
    const int g = of[s], begin = begin_of(s), e = groups + s;
    if (begin) {
      o.shared_n = count(rows[g], chunk);
      o.shared_slot = low[g] && o.shared_n == 1 ? -1 : slot_of(before[g]);
      o.shared_step = runs_of(g) * (a.cols / kCols);
      o.col = (s - starts[g]) * group;
    }
    o.n = (before[e + 1] - before[e]) / parts;
    o.slot = begin == 0 && o.n == 1 ? -1 : slot_of(before[e]);
    return o;
  }
  // The last of n ascending values that is <= x, or -1.
  __device__ static int find(const int* at, int n, int x) {
    int lo = -1, hi = n;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (at[mid] <= x) lo = mid;
      else hi = mid;
    }
    return lo;
  }
};

// The plan by a block, its arrays in `mem`.
__device__ __forceinline__ Plan make_plan(const PagedArgs& a, int* mem) {
  constexpr int threads = kPlanThreads, waves = threads / 64;
  __shared__ int64_t sums[waves];
  __shared__ int scans[waves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n_seq = a.n_seq;
  Plan p{a, mem};
  p.of = p.keys + n_seq;
  p.starts = p.of + n_seq;
  p.rows = p.starts + a.groups + 1;
  p.low = p.rows + a.groups;
  p.high = p.low + a.groups;
  p.live = p.high + a.groups;
  p.before = p.live + a.groups;
  p.group = a.heads / a.kv_heads;
  p.parts = (p.group + kCols - 1) / kCols;
  for (int s = tid; s < n_seq; s += threads) p.keys[s] = a.lens[s] < 0 ? -1 : paged_keys(a, s);  // -1: idle
  int descends = 0;  // groups whose starts do not ascend would overlap: none is one
  for (int g = tid; g <= a.groups && a.groups; g += threads) {
    const int64_t start = a.cu_g[g], next = a.cu_g[min(g + 1, a.groups)];
    p.starts[g] = static_cast<int>(within(start, 0, n_seq));
    if (g == a.groups) break;
    descends |= start > next;
    p.rows[g] = static_cast<int>(within(a.shared[g], 0, 1 << 30));
    p.low[g] = 0x7FFFFFFF;
    p.high[g] = 0;
    p.live[g] = 0x7FFFFFFF;
  }
  p.groups = __syncthreads_or(descends) ? 0 : a.groups;
  // the first of a group's live sequences, the fewest and most keys of them; a wave of one group asks once
  for (int s0 = tid & ~63; s0 < n_seq; s0 += threads) {
    const int s = s0 + lane;
    int g = -1, lo = 0x7FFFFFFF, hi = 0, first = 0x7FFFFFFF;
    if (s < n_seq) {
      g = Plan::find(p.starts, p.groups, s);
      if (g >= 0 && s >= p.starts[g + 1]) g = -1;
      p.of[s] = g;
      if (p.keys[s] >= 0) {
        lo = hi = p.keys[s];
        first = s;
      }
    }
    const int one = __builtin_amdgcn_readfirstlane(g);
    if (__builtin_amdgcn_ballot_w64(g == one) == __builtin_amdgcn_ballot_w64(true)) {
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        lo = min(lo, __shfl_xor(lo, o));
        hi = max(hi, __shfl_xor(hi, o));
        first = min(first, __shfl_xor(first, o));
      }
      if (lane != 0) g = -1;
    }
    if (g >= 0) {
      atomicMin(&p.low[g], lo);
      atomicMax(&p.high[g], hi);
      atomicMin(&p.live[g], first);
    }
  }
  __syncthreads();
  int64_t work = 0;
  for (int g = tid; g < p.groups; g += threads) {
    const int low = Plan::made(&p.low[g]), high = Plan::made(&p.high[g]);
    const int most = p.starts[g + 1] - p.starts[g] > 1 && high > 0 ? min(p.rows[g], low) : 0, whole = most == high;
    p.rows[g] = whole ? most : most & ~(kTileKeys - 1);
    p.low[g] = whole;
    work += static_cast<int64_t>(p.rows[g]) * p.runs_of(g);
  }
  if (p.groups) __syncthreads();
  for (int s = tid; s < n_seq; s += threads) work += static_cast<int64_t>(max(p.keys[s] - p.begin_of(s), 0)) * p.parts;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) work += __shfl_xor(work, o);
  if (lane == 0) sums[wave] = work;
  __syncthreads();
  work = 0;
  for (int w = 0; w < waves; ++w) work += sums[w];
  // (rounded up past what fp32 may lose of it: a chunk is no less than its share)
  const float share = static_cast<float>(work) * 1.000001f / static_cast<float>(a.want);
  p.chunk = (static_cast<uint32_t>(fminf(share, 1 << 30)) / a.unit + 1) * a.unit;
  // pieces of the groups, then of the sequences; one without keys has one, for its zeros
  p.total = 0;
  for (int e0 = 0; e0 < p.groups + n_seq; e0 += threads) {
    const int e = e0 + tid, s = e - p.groups;
    int n = 0;
    if (s < 0) n = Plan::count(p.rows[e], p.chunk) * p.runs_of(e);
    else if (s < n_seq) n = max(Plan::count(max(p.keys[s] - p.begin_of(s), 0), p.chunk), p.begin_of(s) == 0 ? 1 : 0) * p.parts;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(sum, o);
      if (lane >= o) sum += x;
    }
    if (e0) __syncthreads();
    if (lane == 63) scans[wave] = sum;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < waves; ++w) {
      if (w < wave) sum += scans[w];
      all += scans[w];
    }
    if (s < n_seq) p.before[e] = p.total + sum - n;
    p.total += all;
  }
  if (tid == 0) p.before[p.groups + n_seq] = p.total;
  __syncthreads();
  p.total = min(p.total, a.most);
  return p;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PagedArgs a) {
  __shared__ int local[plan_words(kPlanLds, kPlanLds)];
  Owner* owners = owners_of(a);
  const Plan p = make_plan(a, a.n_seq <= kPlanLds && a.groups <= kPlanLds ? local : reinterpret_cast<int*>(owners + a.n_seq));
  for (int at = threadIdx.x; at < p.total; at += kPlanThreads) pieces_of(a)[at] = p.piece(at);
  for (int s = threadIdx.x; s < a.n_seq; s += kPlanThreads) owners[s] = p.owner(s);
  if (threadIdx.x == 0) a.plan[0] = p.total;
}

// The same plan by a wave: lane s has sequence s, and for its group the numbers of its first sequence's lane.
constexpr int kWavePlan = 64;
struct WavePlan {
  int keys, start, members;       // the lane's sequence; its group's first one (itself: none)
  int rows, whole, shared_n;      // its group's shared rows, whether they are all, and their pieces a run
  int n, shared_before, before;   // its own pieces a run; pieces up to the end of its group's (in the first lane), and of its own
  int of_groups, total;           // (in every lane)

  __device__ __forceinline__ static int lane_of(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
  __device__ __forceinline__ void make(const PagedArgs& a, int lane) {
    const int group = a.heads / a.kv_heads, parts = (group + kCols - 1) / kCols;
    int64_t len = -1, begin = 0, end = 0, want = 0;
    if (lane < a.n_seq) len = a.lens[lane];
    if (lane < a.groups) {
      begin = a.cu_g[lane];
      end = a.cu_g[lane + 1];
      want = a.shared[lane];
    }
    keys = static_cast<int>(within(len, -1, static_cast<int64_t>(a.width) << a.page_shift));
    start = lane;
    members = 1;
    rows = whole = shared_n = 0;
    // (groups whose starts do not ascend would overlap: none is one)
    if (a.groups && !__builtin_amdgcn_ballot_w64(begin > end)) {
      const int b = static_cast<int>(within(begin, 0, a.n_seq)), e = static_cast<int>(within(end, b, a.n_seq));
      // a group of several tells its first sequence's lane its number; the others look there
      const int told = __builtin_amdgcn_ds_permute(4 * (e - b > 1 ? b : 63), e - b > 1 ? lane + 1 : 0);
      // (lane 63 begins no group of several, so what the others tell it is nothing)
      const uint64_t firsts = __builtin_amdgcn_ballot_w64(told > 0 && lane < 63) & (~uint64_t{0} >> (63 - lane));
      const int first = firsts ? 63 - __builtin_clzll(firsts) : lane, g = __shfl(told, first) - 1;
      const int last = __shfl(e, max(g, 0)), most = __shfl(static_cast<int>(within(want, 0, 1 << 30)), max(g, 0));
      const bool in = firsts && lane < last;
      if (in) {
        start = first;
        members = last - first;
      }
      int low = keys < 0 ? 0x7FFFFFFF : keys, high = max(keys, 0);
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(low, o), y = __shfl_up(high, o);
        if (lane - o >= start) {
          low = min(low, x);
          high = max(high, y);
        }
      }
      low = __shfl(low, start + members - 1);
      high = __shfl(high, start + members - 1);
      if (in && high > 0) {
        const int have = min(most, low);
        whole = have == high;
        rows = whole ? have : have & ~(kTileKeys - 1);
      }
    }
    const int mine = max(keys - rows, 0), runs = (members * group + a.cols - 1) / a.cols;
    const float work = static_cast<float>(mine) * parts + (lane == start ? static_cast<float>(rows) * runs : 0.f);
    const float share = group_sum<64>(work) * 1.0001f / static_cast<float>(a.want);  // (no less than its share)
    const uint32_t chunk = (static_cast<uint32_t>(fminf(share, 1 << 30)) / a.unit + 1) * a.unit;
    shared_n = Plan::count(rows, chunk);
    n = lane < a.n_seq ? max(Plan::count(mine, chunk), rows == 0 ? 1 : 0) : 0;
    shared_before = wave_scan(lane == start ? shared_n * runs : 0);
    of_groups = lane_of(shared_before, 63);
    before = of_groups + wave_scan(n * parts);
    total = min(lane_of(before, 63), a.most);
  }
  // (every lane asks for the same piece)
  __device__ __forceinline__ Piece piece(const PagedArgs& a, int at) const {
    const int group = a.heads / a.kv_heads, parts = (group + kCols - 1) / kCols, tiles = a.cols / kCols;
    if (at < of_groups) {
      const int s = __builtin_ctzll(__builtin_amdgcn_ballot_w64(shared_before > at));
      const int columns = lane_of(members, s) * group, runs = (columns + a.cols - 1) / a.cols;
      const int k = lane_of(rows, s), pieces = lane_of(shared_n, s);
      const int x = at - (lane_of(shared_before, s) - pieces * runs), i = x / runs, r = x % runs, size = Plan::size_of(k, pieces);
      const int live = s + __builtin_ctzll(__builtin_amdgcn_ballot_w64(keys >= 0) >> s);  // (shared rows are those of live ones)
      return Piece{s, r * a.cols, min(a.cols, columns - r * a.cols), i * size, min((i + 1) * size, k),
                   lane_of(whole, s) && pieces == 1 ? -1 : at * tiles, live, 0};
    }
    const int s = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before > at)), pieces = lane_of(n, s), begin = lane_of(rows, s);
    const int mine = max(lane_of(keys, s) - begin, 0), x = at - (lane_of(before, s) - pieces * parts), i = x / parts, r = x % parts;
    const int size = Plan::size_of(mine, pieces);
    return Piece{s, r * kCols, min(kCols, group - r * kCols), begin + i * size, begin + min((i + 1) * size, mine),
                 begin == 0 && pieces == 1 ? -1 : of_groups * tiles + (at - of_groups), s, 0};
  }
  // Of the lane's own sequence.
  __device__ __forceinline__ Owner owner(const PagedArgs& a, int lane) const {
    const int group = a.heads / a.kv_heads, parts = (group + kCols - 1) / kCols, tiles = a.cols / kCols;
    const int runs = (members * group + a.cols - 1) / a.cols, end = __shfl(shared_before, start);
    Owner o{};
    if (rows) {
      o.shared_n = shared_n;
      o.shared_slot = whole && shared_n == 1 ? -1 : (end - shared_n * runs) * tiles;
      o.shared_step = runs * tiles;
      o.col = (lane - start) * group;
    }
    o.n = n;
    o.slot = rows == 0 && n == 1 ? -1 : of_groups * tiles + (before - n * parts - of_groups);
    return o;
  }
};

// The queries of 16 columns from `col` on of the sequences from `seq` on; columns past the last of `cols` repeat it.
template <class T, int D>
__device__ __forceinline__ void paged_queries(const PagedArgs& a, int seq, int col, int cols, int kvh, int lane,
                                              typename Types<T>::v8 (&q)[D / 32]) {
  typedef typename Types<T>::v8 v8;
  const int group = a.heads / a.kv_heads, x = col + min(lane & 15, cols - 1);
  const T* at = static_cast<const T*>(a.q) + (seq + x / group) * a.q_row + (kvh * group + x % group) * a.q_head + 8 * (lane >> 4);
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    q[j] = *reinterpret_cast<const v8*>(at + 32 * j);
    if (a.scale < 0.f) q[j] = -q[j];  // scores are scaled by a positive factor after the product
  }
}
// 0: the smallest number instead; a hidden score (-infinity) times zero would be NaN.
__device__ __forceinline__ float paged_factor(const PagedArgs& a) { return fmaxf(__builtin_fabsf(a.scale) * kLog2e, __FLT_DENORM_MIN__); }

// A wave's results of its first `cols` columns to part `part`.
template <class T, int D>
__device__ __forceinline__ void paged_hand_in(const PagedMerge<D>& x, const PagedState<T, D, 1>& st, int part, int cols, int lane) {
  const int i = lane & 15, g = lane >> 4;
  const float l = xor_add<32>(xor_add<16>(st.l[0]));
  if (i >= cols) return;
  if (g == 0) {
    x.m[part * kCols + i] = st.m[0];
    x.l[part * kCols + i] = l;
  }
  float* to = x.acc + (part * x.cols + i) * PagedMerge<D>::kPitch + 4 * g;
#pragma unroll
  for (int db = 0; db < D / 16; ++db) *reinterpret_cast<f4v*>(to + 16 * db) = st.o[0][db];
}

// The sum over the parts for column col and dims d .. d + 3: o and l relative to exp2(m).
template <int D>
__device__ __forceinline__ f4v paged_sum(const PagedMerge<D>& x, int parts, int col, int d, float& m, float& l) {
  m = -INFINITY;
  l = 0.f;
  f4v o = {};
  for (int w = 0; w < parts; ++w) m = fmaxf(m, x.m[w * kCols + col]);
  for (int w = 0; w < parts; ++w) {
    const float mw = x.m[w * kCols + col], f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - m);
    l = fmaf(f, x.l[w * kCols + col], l);
    o += f * *reinterpret_cast<const f4v*>(x.acc + (w * x.cols + col) * PagedMerge<D>::kPitch + d);
  }
  return o;
}

// Four dims of a column, or zeros: nothing was seen. (An idle sequence of a group sees nothing, whatever its group sees.)
template <class T>
__device__ __forceinline__ void paged_store(const PagedArgs& a, int seq, int head, int d, const f4v& o, float l) {
  typedef T v4 __attribute__((ext_vector_type(4)));
  const bool none = l == 0.f || a.lens[seq] <= 0;
  v4 y;
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = static_cast<T>(none ? 0.f : o[r] / l);
  *reinterpret_cast<v4*>(static_cast<T*>(a.out) + seq * a.o_row + head * a.o_head + d) = y;
}

// A piece of at most 16 columns: its tiles in turn to the block's waves, as many as there are tiles.
template <class T, int D>
__device__ __forceinline__ void paged_piece(const PagedArgs& a, const Piece& p, int kvh, const int32_t* table, float* lds) {
  const int waves = blockDim.x / 64, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = a.heads / a.kv_heads, parts = min(waves, (p.end - p.begin + kTileKeys - 1) / kTileKeys);
  const PagedMerge<D> x(lds, waves, p.cols);
  if (wave < parts) {
    typename Types<T>::v8 q[1][D / 32];
    paged_queries<T, D>(a, p.seq, p.col, p.cols, kvh, lane, q[0]);
    PagedState<T, D, 1> st;
    paged_tiles<T, D, 1>(a, table, kvh, p.begin / kTileKeys + wave, waves, p.end, q, paged_factor(a), lane, st);
    paged_hand_in<T, D>(x, st, wave, p.cols, lane);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.cols * (D / 4); e += blockDim.x) {
    const int col = e / (D / 4), d = e % (D / 4) * 4;
    float m, l;
    const f4v o = paged_sum<D>(x, parts, col, d, m, l);
    if (p.slot < 0) {
      paged_store<T>(a, p.seq + (p.col + col) / group, kvh * group + (p.col + col) % group, d, o, l);
    } else {
      const int64_t at = (static_cast<int64_t>(p.slot) * a.kv_heads + kvh) * kCols + col;
      *reinterpret_cast<f4v*>(a.part + at * D + d) = o;
      if (d == 0) reinterpret_cast<float2*>(a.ml)[at] = make_float2(m, l);
    }
  }
}

// A piece of many columns: wave w has columns 16 CT w .. and all of the keys, which arrive in LDS by direct copies, a ring of
// kStages steps of two tiles, so that a row of K and V is read once for 64 CT columns. A tile of a page is contiguous, V's just as
// the operands are read; K's 16-byte chunks are swapped within a row so that the 16 rows of a read lie in different banks.
// Bound by what every block pays once (plan, first tiles, results: about 12 us) and then by the LDS reads, 32 KB a wave and step:
// 64 answers x 4 heads over 8000 shared rows of 8 heads of 128 take 20 us with the plan, each further 8000 rows 10 (0.84 PFLOP/s); waves
// that share out the keys instead, 32 columns each, took 62. Steps of one tile, four stages: 2% more.
constexpr int kStages = 2, kWaves = 4, kStep = 2;
template <int D>
__device__ __forceinline__ int wide_swap(int row) {
  return D == 128 ? (row & 3) | ((row >> 3) & 3) << 2 : ((row >> 1) & 1) | ((row >> 3) & 3) << 1;
}

// A step's keys: K at LDS address k, V at v, a tile kTile bytes on from the other. MASKED: left[t] of the lane's 8 keys of tile t count.
template <class T, int D, int CT, bool MASKED>
__device__ __forceinline__ void wide_step(uint32_t k, uint32_t v, const typename Types<T>::v8 (&q)[CT][D / 32], float factor,
                                          const int (&left)[kStep], PagedState<T, D, CT>& st) {
  typedef typename Types<T>::v8 v8;
  typedef typename Types<T>::v2 v2;
  typedef __attribute__((address_space(3))) v8 lds_v8;
  constexpr uint32_t kRowBytes = 2 * D, kTile = kTileKeys * kRowBytes;
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  f4v s[CT][kStep][2];
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int t = 0; t < kStep; ++t) s[c][t][0] = s[c][t][1] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    const uint32_t at = k + ((4 * j + g) ^ wide_swap<D>(8 * (i >> 2) + (i & 3))) * 16;
    v8 x[kStep][2];
#pragma unroll
    for (int t = 0; t < kStep; ++t)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) x[t][kt] = *reinterpret_cast<lds_v8*>(static_cast<uintptr_t>(at + t * kTile + 4 * kt * kRowBytes));
#pragma unroll
    for (int t = 0; t < kStep; ++t)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int c = 0; c < CT; ++c) s[c][t][kt] = mfma16(x[t][kt], q[c][j], s[c][t][kt]);
  }
  v8 p[CT][kStep];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < kStep; ++t)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (MASKED && 4 * kt + r >= left[t]) s[c][t][kt][r] = -INFINITY;
          top = __builtin_elementwise_maximum(top, s[c][t][kt][r]);
        }
    top = fmaf(xor_max<32>(xor_max<16>(top)), factor, -Types<T>::kLift);
    if (__builtin_amdgcn_ballot_w64(top > st.m[c] + Types<T>::kSlack)) {
      const float m_new = fmaxf(st.m[c], top), corr = st.m[c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m[c] - m_new);
      st.l[c] *= corr;
#pragma unroll
      for (int db = 0; db < D / 16; ++db) st.o[c][db] *= corr;
      st.m[c] = m_new;
    }
    const float m = st.m[c] == -INFINITY ? 0.f : st.m[c];
    float sum[kStep] = {};
#pragma unroll
    for (int t = 0; t < kStep; ++t)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          v2 x;
          x[0] = static_cast<T>(__builtin_amdgcn_exp2f(fmaf(s[c][t][kt][r], factor, -m)));
          x[1] = static_cast<T>(__builtin_amdgcn_exp2f(fmaf(s[c][t][kt][r + 1], factor, -m)));
          sum[t] = add_pair(x, sum[t]);
          p[c][t][4 * kt + r] = x[0];
          p[c][t][4 * kt + r + 1] = x[1];
        }
    st.l[c] += sum[0] + sum[1];
  }
#pragma unroll
  for (int t = 0; t < kStep; ++t)
#pragma unroll
    for (int db = 0; db < D / 16; ++db) {
      v8 x = *reinterpret_cast<lds_v8*>(static_cast<uintptr_t>(v + t * kTile + (g * D + i) * 16 + db * 256));
      if constexpr (MASKED) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e >= left[t]) x[e] = static_cast<T>(0.f);
      }
#pragma unroll
      for (int c = 0; c < CT; ++c) st.o[c][db] = mfma16(x, p[c][t], st.o[c][db]);
    }
}

template <class T, int D, int CT>
__device__ __forceinline__ void paged_wide(const PagedArgs& a, const Piece& p, int kvh, const int32_t* table, float* lds) {
  typedef typename Types<T>::v8 v8;
  constexpr int kTile = kTileKeys * D * 2, kStage = 2 * kStep * kTile;  // bytes of a tile of K or V, of a step of both
  constexpr int kCopies = kTile / 1024 / kWaves;                        // of a tile of K, and of V, a wave
  constexpr int kRowBytes = 2 * D, kCopyRows = 1024 / kRowBytes;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, g = lane >> 4, group = a.heads / a.kv_heads, col0 = kCols * CT * wave;
  const bool live = col0 < p.cols;
  const uint32_t ring = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  const int first = p.begin / kTileKeys, tiles = (p.end + kTileKeys - 1) / kTileKeys - first, rows = 1 << a.page_shift;
  const int steps = (tiles + kStep - 1) / kStep;
  PagedPages pages = paged_pages(a, table, first + lane, p.end);
  uint32_t ok = 0;  // two bits a tile of the ring: the pages of its halves
  const auto issue = [&](int n) {
    const int s = n % kStages;
#pragma unroll
    for (int t = 0; t < kStep; ++t) {  // (a tile past the end has no page: page 0 is copied, and none of it counts)
      const int x = kStep * n + t, place = 2 * (kStep * s + t);
      if (t == 0 && x && (x & 63) == 0) pages = paged_pages(a, table, first + x + lane, p.end);
      const int lo = __builtin_amdgcn_readlane(pages.lo, x & 63), hi = __builtin_amdgcn_readlane(pages.hi, x & 63);
      ok = (ok & ~(3u << place)) | static_cast<uint32_t>((lo >= 0) | (hi >= 0) << 1) << place;
      const uint32_t to = ring + s * kStage + t * kTile;
      const int row = ((first + x) * kTileKeys) & (rows - 1);
      const int64_t at_lo = ((static_cast<int64_t>(max(lo, 0)) * a.kv_heads + kvh) * rows + row) * kRowBytes;
      // (a page of 16 rows: the second half begins another page's rows)
      const int64_t other = (static_cast<int64_t>(max(hi, 0)) * a.kv_heads + kvh) * rows * kRowBytes - kTile / 2;
      const int64_t at_hi = a.page_shift == 4 ? other : at_lo;
#pragma unroll
      for (int c = 0; c < kCopies; ++c) {
        const int blk = kCopies * wave + c, r = blk * kCopyRows + lane / (D / 8), chunk = (lane % (D / 8)) ^ wide_swap<D>(r);
        const int64_t at = blk * 1024 < kTile / 2 ? at_lo : at_hi;
        dma16_s(static_cast<uint32_t>(r * kRowBytes + chunk * 16), static_cast<const uint8_t*>(a.k) + at, to + blk * 1024);
        dma16_s(static_cast<uint32_t>(blk * 1024 + lane * 16), static_cast<const uint8_t*>(a.v) + at, to + kStep * kTile + blk * 1024);
      }
    }
  };
#pragma unroll
  for (int n = 0; n < kStages - 1; ++n)
    if (n < steps) issue(n);
  v8 q[CT][D / 32];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int col = min(col0 + kCols * c, p.cols - 1);  // (a wave without columns has the last one's)
    paged_queries<T, D>(a, p.seq, p.col + col, p.cols - col, kvh, lane, q[c]);
  }
  const float factor = paged_factor(a);
  PagedState<T, D, CT> st;
#pragma unroll
  for (int c = 0; c < CT; ++c) {
#pragma unroll
    for (int db = 0; db < D / 16; ++db) st.o[c][db] = f4v{0.f, 0.f, 0.f, 0.f};
    st.m[c] = -INFINITY;
    st.l[c] = 0.f;
  }
  for (int n = 0; n < steps; ++n) {
    // step n visible to every wave, every one done with step n - 1, whose place step n + kStages - 1 takes
    wait_stages_ahead<2 * kStep * kCopies, kStages - 1>(min(kStages - 2, steps - 1 - n));
    lds_barrier();
    const uint32_t at = ring + n % kStages * kStage, has = (ok >> (2 * kStep * (n % kStages))) & 15;
    if (n + kStages - 1 < steps) issue(n + kStages - 1);
    if (!live) continue;
    const int end = p.end - (first + kStep * n) * kTileKeys;
    const uint32_t k = at + (8 * (i >> 2) + (i & 3)) * kRowBytes, v = at + kStep * kTile;
    const int left[kStep] = {has >> (lane >> 5) & 1 ? end - 8 * g : 0, has >> (2 + (lane >> 5)) & 1 ? end - kTileKeys - 8 * g : 0};
    if (end >= kStep * kTileKeys && has == 15) wide_step<T, D, CT, false>(k, v, q, factor, left, st);
    else wide_step<T, D, CT, true>(k, v, q, factor, left, st);
  }
  if (!live) return;
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const float l = xor_add<32>(xor_add<16>(st.l[c]));
    const int col = col0 + kCols * c + i;
    if (col >= p.cols) continue;
    if (p.slot < 0) {
      const int seq = p.seq + (p.col + col) / group, head = kvh * group + (p.col + col) % group;
#pragma unroll
      for (int db = 0; db < D / 16; ++db) paged_store<T>(a, seq, head, 16 * db + 4 * g, st.o[c][db], l);
    } else {
      const int64_t to = (static_cast<int64_t>(p.slot + col / kCols) * a.kv_heads + kvh) * kCols + i;
      if (g == 0) *reinterpret_cast<float2*>(a.ml + 2 * to) = make_float2(st.m[c], l);
#pragma unroll
      for (int db = 0; db < D / 16; ++db) *reinterpret_cast<f4v*>(a.part + to * D + 16 * db + 4 * g) = st.o[c][db];
    }
  }
}

// CT < 0: a block for each sequence, key/value head and 16 of its columns. Else a block for each piece and key/value head; CT > 0:
// those of more than 16 columns are wide.
template <class T, int D, int CT>
__global__ void __launch_bounds__(CT < 0 ? 512 : 64 * kWaves, 2) paged_attention_kernel(PagedArgs a) {
  extern __shared__ __align__(1024) float lds[];
  const int kvh = blockIdx.x % a.kv_heads;
  const unsigned at = blockIdx.x / a.kv_heads;
  if constexpr (CT < 0) {
    const int group = a.heads / a.kv_heads, parts = (group + kCols - 1) / kCols;
    const int col = static_cast<int>(at % parts) * kCols, seq = static_cast<int>(at / parts);
    const Piece p{seq, col, min(kCols, group - col), 0, paged_keys(a, seq), -1, seq, 0};
    paged_piece<T, D>(a, p, kvh, a.table + static_cast<int64_t>(seq) * a.width, lds);
  } else {
    Piece p;
    if (a.n_seq <= kWavePlan && a.groups <= kWavePlan) {
      WavePlan plan;
      plan.make(a, threadIdx.x & 63);
      if (blockIdx.x == 0 && static_cast<int>(threadIdx.x) < a.n_seq) owners_of(a)[threadIdx.x] = plan.owner(a, threadIdx.x);
      if (static_cast<int>(at) >= plan.total) return;
      p = plan.piece(a, at);
    } else {
      if (static_cast<int>(at) >= a.plan[0]) return;
      p = pieces_of(a)[at];
    }
    const int32_t* table = a.table + static_cast<int64_t>(p.table) * a.width;
    if constexpr (CT > 0) {
      if (p.cols > kCols) {
        paged_wide<T, D, CT>(a, p, kvh, table, lds);
        return;
      }
    }
    paged_piece<T, D>(a, p, kvh, table, lds);
  }
}

// Joins what the pieces of a sequence left for a query head: W waves a head, each every W-th piece, a lane a piece's (m, l) and D /
// 64 dims. What a wave needs is on its way before the weights are known. Bound by latency.
template <class T, int D, int W>
__global__ void __launch_bounds__(256) paged_combine_kernel(PagedArgs a) {
  constexpr int kDims = D / 64, kBatch = 8;
  typedef float dims __attribute__((ext_vector_type(kDims)));
  __shared__ float lds[W > 1 ? W : 1][64][kDims + 2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % W;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (4 / W) + wave / W;
  const int seq = static_cast<int>(at / a.heads), head = static_cast<int>(at % a.heads);
  if (seq >= a.n_seq) return;  // (W = 1)
  const Owner o = owners_of(a)[seq];
  const int n = o.shared_n + o.n, group = a.heads / a.kv_heads, kvh = head / group, col = head % group, step = (group + kCols - 1) / kCols;
  if ((o.shared_n == 0 || o.shared_slot < 0) && (o.n == 0 || o.slot < 0)) return;  // its block finished it
  const auto slot = [&](int i) {
    const bool shared = i < o.shared_n;
    const int c = shared ? o.col + col : col, first = shared ? o.shared_slot + i * o.shared_step : o.slot + (i - o.shared_n) * step;
    return (static_cast<int64_t>(first + c / kCols) * a.kv_heads + kvh) * kCols + c % kCols;
  };
  float m = -INFINITY, l = 0.f;
  dims y = {};
  for (int i0 = part; i0 < n; i0 += 64 * W) {
    const int here = min(64, (n - i0 + W - 1) / W);  // pieces of this round: i0, i0 + W, ..
    dims x[kBatch];
    const auto load = [&](int j0) {  // past the end the last one
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        x[j] = *reinterpret_cast<const dims*>(a.part + slot(i0 + W * min(j0 + j, here - 1)) * D + kDims * lane);
    };
    load(0);
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < here) ml = reinterpret_cast<const float2*>(a.ml)[slot(i0 + W * lane)];
    const float top = fmaxf(m, group_max<64>(ml.x)), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    const float w = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - top);
    l = fmaf(l, f, group_sum<64>(w * ml.y));
    y *= f;
    m = top;
    for (int j0 = 0;;) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (j0 + j < here) y += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), j0 + j)) * x[j];
      j0 += kBatch;
      if (j0 >= here) break;
      load(j0);
    }
  }
  if constexpr (W > 1) {
    float* mine = lds[wave][lane];
    mine[0] = m;
    mine[1] = l;
#pragma unroll
    for (int d = 0; d < kDims; ++d) mine[2 + d] = y[d];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int i = 1; i < W; ++i) m = fmaxf(m, lds[i][lane][0]);
    const float f = mine[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine[0] - m);
    l *= f;
    y *= f;
#pragma unroll
    for (int i = 1; i < W; ++i) {
      const float* other = lds[i][lane];
      const float w = other[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(other[0] - m);
      l = fmaf(w, other[1], l);
#pragma unroll
      for (int d = 0; d < kDims; ++d) y[d] = fmaf(w, other[2 + d], y[d]);
    }
  }
  typedef T out __attribute__((ext_vector_type(kDims)));
  out z;
#pragma unroll
  for (int d = 0; d < kDims; ++d) z[d] = static_cast<T>(l == 0.f || a.lens[seq] <= 0 ? 0.f : y[d] / l);
  *reinterpret_cast<out*>(static_cast<T*>(a.out) + seq * a.o_row + head * a.o_head + kDims * lane) = z;
}

// What of a call goes by sizes alone (the lengths are on the device).
struct PagedSizes {
  int cols, want, waves, direct_waves;
  int64_t most, slots, ints, floats;  // pieces, 16-column results, the plan's words, workspace
};
// Short tables are not cut up: a block takes a sequence whole, and reads rows that it shares as the others do, which the last-level
// caches bear. Up to 1024 rows, 768 for few sequences with heads of 128, and 2048 for many of which none shares (us whole / cut: 1 x 20
// heads of 64 over 600 rows 5.9 / 9.1, 1000 7.7 / 9.1, 1500 9.7 / 9.2; 1 x 8 heads of 128 over 600 8.7 / 10.5, 1000 12.3 / 10.7; 16 x
// 20 over 1500 27.8 / 31.2; 64 x 8 of 128 over 2000 91 / 95; 8 groups of 5 x 20 over 400 shared and 100 own rows 11.3 / 13.9, 1000
// shared 14.4 / 12.9). How many sequences a group has is on the device: a call captured once lists as many groups as it may ever have,
// most of them empty, so as many groups as sequences are groups too (8 x 5 beams over 1500 rows, as 40 groups: 14.7 us, taken as none
// 22.8; 64 answers to 8000 rows, as 64: 36.6 and 217; but 17 x 20 heads over 1500 rows that share nothing 32.5 and 28.9 when they are
// called 17 groups, 64 x 8 of 128 over 2000 94 and 91).
// Else the keys make about 512 blocks' pieces, one or two a CU at a time (the 17 long sequences above with 256 / 512 / 768 / 1024: 96 /
// 87 / 93 / 90 us), half as many where a group's columns are 65 to 256, whose results cost as much as keys (us with half / all, 8 heads
// of 128: 80 columns over 8000 rows 21.7 / 25.2, 128 22.6 / 26.3, 192 28.7 / 29.6, 256 31.5 / 32.7, and 64 answers above 34.0 / 36.3;
// over 2000 15.7 / 15.2, 16.3 / 17.6, 17.5 / 22.2, 19.7 / 21.1; but over 40000 62 / 59, 63 / 57, 84 / 69, 101 / 85). Groups of more
// than 16 columns go by 64 at a time, of more than 256 by 128 (us by 64 / 128: 256 columns over 8000 rows 34.0 / 35.6, 512 over 30000
// 109 / 99). Where any group could have more than 16 columns the launch is ready for 64, which costs smaller ones nothing (8 x 5 beams
// 14.7 us by either); 128, and half the pieces, go by the average of as many groups as the call names. The joining launch has a wave a
// query head where there are 512 of them and more (800: 15.6 us a call, with four 16.4; 20: 9.9 and 9.1).
constexpr int kDirectRows = 1024, kDirectMany = 2048, kDirectFew = 768, kManyItems = 128, kWantBlocks = 512, kManyHeads = 512;

int merge_bytes(int dim, int waves, int cols) {
  return dim == 64 ? PagedMerge<64>::bytes(waves, cols) : PagedMerge<128>::bytes(waves, cols);
}

PagedSizes paged_sizes(int n_seq, int heads, int kv_heads, int64_t capacity, int groups, int dim) {
  PagedSizes p = {};
  const int64_t group = heads / kv_heads, parts = (group + kCols - 1) / kCols;
  p.direct_waves = static_cast<int>(std::min<int64_t>(8, (capacity + kTileKeys - 1) / kTileKeys));
  while (merge_bytes(dim, p.direct_waves, static_cast<int>(std::min<int64_t>(kCols, group))) > 65536) --p.direct_waves;
  p.waves = kWaves;
  if (n_seq == 1) groups = 0;
  const bool many_items = static_cast<int64_t>(n_seq) * kv_heads * parts >= kManyItems;
  if (capacity <= (many_items ? groups ? kDirectRows : kDirectMany : dim == 64 ? kDirectRows : kDirectFew)) {
    p.floats = 4;
    return p;
  }
  const int64_t columns = groups ? (n_seq + groups - 1) / groups * group : 0;  // of an average group
  p.cols = columns > 256 ? 128 : groups && n_seq * group > kCols ? 64 : kCols;
  p.want = std::max(1, (columns > 64 && columns <= 256 ? kWantBlocks / 2 : kWantBlocks) / kv_heads);
  // each run of columns has the pieces that fill its share of `want`, and one more
  const int64_t runs = groups ? n_seq * group / p.cols + std::min(groups, n_seq / 2) : 0;
  p.most = p.want + runs + n_seq * parts + 1;
  p.slots = p.cols / kCols * (p.want + runs) + n_seq * parts + 1;
  p.ints = 4 + 8 * p.most + 8 * static_cast<int64_t>(n_seq) + (n_seq <= kPlanLds && groups <= kPlanLds ? 0 : plan_words(n_seq, groups));
  p.ints = (p.ints + 3) / 4 * 4;
  p.floats = p.ints + p.slots * kv_heads * kCols * (dim + 2);
  return p;
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool rows_ok(const void* p, int64_t row, int64_t head) { return aligned(p, 16) && row % 8 == 0 && head % 8 == 0; }

// What every call asks of its sizes; FW_OK or FW_EINVAL.
int check_paged(int n_seq, int heads, int kv_heads, int width, int page, int groups, int head_dim) {
  const char* what = "decode_attention_paged";
  if (page_shift_of(page) < 0) return fw_fail(FW_EINVAL, "%s: page must be 16, 32, 64, 128 or 256 rows", what);
  if (head_dim != 64 && head_dim != 128) return fw_fail(FW_EINVAL, "%s: head_dim must be 64 or 128", what);
  if (n_seq <= 0 || width <= 0 || groups < 0) return fw_fail(FW_EINVAL, "%s: n_seq and width must be positive, groups not negative", what);
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads) return fw_fail(FW_EINVAL, "%s: heads must be a multiple of kv_heads", what);
  if (static_cast<int64_t>(width) * page > (1 << 30)) return fw_fail(FW_EINVAL, "%s: at most 2^30 rows a sequence", what);
  if (n_seq > 65535 || groups > 65535) return fw_fail(FW_EINVAL, "%s: too many sequences", what);
  if (heads > (1 << 14)) return fw_fail(FW_EINVAL, "%s: too many heads", what);  // columns of a group in 32 bits
  return FW_OK;
}

}  // namespace
}  // namespace fw

using namespace fw;

extern "C" int64_t fw_decode_attention_paged_ws_floats(int n_seq, int heads, int kv_heads, int width, int page, int groups,
                                                       int head_dim) {
  if (check_paged(n_seq, heads, kv_heads, width, page, groups, head_dim)) return 0;
  return paged_sizes(n_seq, heads, kv_heads, static_cast<int64_t>(width) * page, groups, head_dim).floats;
}

extern "C" int fw_decode_attention_paged(const void* q, int64_t q_row, int64_t q_head, const void* k_pages, const void* v_pages,
                                         const int32_t* table, const int64_t* lens, const int64_t* cu_groups,
                                         const int64_t* shared, void* out, int64_t o_row, int64_t o_head, int n_seq, int heads,
                                         int kv_heads, int n_pages, int page, int width, int groups, int head_dim, int dtype,
                                         float scale, float* ws, int64_t ws_floats, hipStream_t stream) {
  const char* what = "decode_attention_paged";
  if (const int rc = check_paged(n_seq, heads, kv_heads, width, page, groups, head_dim)) return rc;
  if (n_pages <= 0) return fw_fail(FW_EINVAL, "%s: n_pages must be positive", what);
  if (dtype != FW_F16 && dtype != FW_BF16) return fw_fail(FW_EINVAL, "%s: dtype must be FW_F16 or FW_BF16", what);
  if (!q || !k_pages || !v_pages || !table || !lens || !out || (groups > 0 && (!cu_groups || !shared)))
    return fw_fail(FW_EINVAL, "%s: null pointer", what);
  if (!(__builtin_fabsf(scale) * kLog2e < INFINITY))
    return fw_fail(FW_EINVAL, "%s: scale must be finite (and below 2.3e38 in size)", what);
  if (!rows_ok(q, q_row, q_head) || !rows_ok(out, o_row, o_head) || !aligned(k_pages, 16) || !aligned(v_pages, 16))
    return fw_fail(FW_EINVAL, "%s: q, out and the pages must be 16-byte aligned with strides in multiples of 8", what);
  const PagedSizes p = paged_sizes(n_seq, heads, kv_heads, static_cast<int64_t>(width) * page, groups, head_dim);
  if (n_seq == 1) groups = 0;
  if (!ws || ws_floats < p.floats || !aligned(ws, 16))
    return fw_fail(FW_EINVAL, "%s: workspace needs %lld floats, 16-byte aligned", what, static_cast<long long>(p.floats));
  const int64_t all = static_cast<int64_t>(heads) * n_seq;
  const bool many = all >= kManyHeads;  // the joining launch has a wave for each, else four
  const int group = heads / kv_heads, parts = (group + kCols - 1) / kCols;
  const int waves = p.most ? p.waves : p.direct_waves, cols = p.cols ? kCols : std::min(kCols, group);
  const int64_t blocks = kv_heads * (p.most ? p.most : static_cast<int64_t>(n_seq) * parts);
  if (!grid_ok(blocks, 64 * waves) || !grid_ok((all + 3) / 4, 256) || p.slots > 0x7FFFFFFF / kCols)
    return fw_fail(FW_EINVAL, "%s: too many sequences", what);
  PagedArgs a{q, k_pages, v_pages, out, q_row, q_head, o_row, o_head, table, lens, cu_groups, shared, n_seq, heads, kv_heads,
              groups, width, n_pages, page_shift_of(page), scale, p.cols, p.want, static_cast<uint32_t>(kTileKeys * p.waves),
              static_cast<int>(p.most), reinterpret_cast<int*>(ws),
              ws + p.ints, nullptr};
  a.ml = a.part + p.slots * kv_heads * kCols * head_dim;
  int lds = merge_bytes(head_dim, waves, cols);
  if (p.cols > kCols) lds = std::max(lds, kStages * kStep * 2 * kTileKeys * head_dim * 2);
  if (p.most && (n_seq > kWavePlan || groups > kWavePlan)) {
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, a);
    if (const int rc = fw_check_launch(what)) return rc;
  }
  const auto run = [&](auto t, auto d) {
    typedef decltype(t) T;
    constexpr int D = decltype(d)::value;
    const auto kernel = !p.most            ? paged_attention_kernel<T, D, -1>
                        : p.cols == kCols ? paged_attention_kernel<T, D, 0>
                        : p.cols == 64    ? paged_attention_kernel<T, D, 1>
                                          : paged_attention_kernel<T, D, 2>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(64 * waves), lds, stream, a);
    if (const int rc = fw_check_launch(what)) return rc;
    if (!p.most) return static_cast<int>(FW_OK);
    const auto combine = many ? paged_combine_kernel<T, D, 1> : paged_combine_kernel<T, D, 4>;
    hipLaunchKernelGGL(combine, dim3(static_cast<unsigned>(many ? (all + 3) / 4 : all)), dim3(256), 0, stream, a);
    return fw_check_launch("decode_attention_paged combine");
  };
  const std::integral_constant<int, 64> d64;
  const std::integral_constant<int, 128> d128;
  if (dtype == FW_F16) return head_dim == 64 ? run(_Float16(), d64) : run(_Float16(), d128);
  return head_dim == 64 ? run(__bf16(), d64) : run(__bf16(), d128);
}
