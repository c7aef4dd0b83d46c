// A key/value cache in pages for gfx950: the pages that sequences hold brought up to their lengths, the slots of new rows,
// and rows written to their slots (layout: pages.h).
#include <algorithm>

#include "packed_rows.h"
#include "pages.h"

namespace fw {
namespace {

// ------------------------------------------------------------------------------------------
// Page map. Sequence s wants the pages of rows 0 .. pos[s] + new - 1 (at most `width`). What it holds beyond them and owns goes
// back onto the stack of free pages, in the order of sequences and entries, then the missing ones are taken off its top in the
// same order: an exclusive sum over the sequences gives each its places, so the result depends on nothing else.
// Bound by latency: one block does all of it in LDS, kTile sequences at a time. The slots are found in the same launch where
// the rows are few, or by further blocks where nothing that the sums are made from is written; else a second launch has a thread for
// each row (64 sequences of a token 4.5 us; 600 of which some bring prompts, 84000 rows, 8.1, in place with two launches 12).
// ------------------------------------------------------------------------------------------
constexpr int kTile = 1024;

struct MapArgs {
  const int64_t *pos, *cu, *held, *own, *count;
  int32_t *table, *stack;
  int64_t *held_out, *count_out, *slots;
  int64_t rows, stack_size;
  int n_seq, width, page_shift;
};

// Sequence s: its first new packed row, and the pages it has, wants (within the table), and needs.
struct MapSeq {
  int64_t begin, pos, need;
  int held, want, low;  // low: entries from here on go back
};

__device__ __forceinline__ MapSeq map_seq(const MapArgs& a, int s) {
  MapSeq x;
  x.begin = within(a.cu[s], 0, a.rows);
  const int64_t end = within(a.cu[s + 1], x.begin, a.rows);
  x.pos = min(a.pos[s], int64_t{1} << 62);  // (sums with it stay positive)
  x.held = static_cast<int>(within(a.held[s], 0, a.width));
  const int64_t page = int64_t{1} << a.page_shift;
  x.need = x.pos < 0 ? x.held : (x.pos + (end - x.begin) + page - 1) >> a.page_shift;
  x.want = static_cast<int>(min(x.need, static_cast<int64_t>(a.width)));
  x.low = max(x.want, a.own ? static_cast<int>(within(a.own[s], 0, a.width)) : 0);
  return x;
}

// Slot of the row `row` of sequence s that holds `held` pages.
__device__ __forceinline__ int64_t map_slot(const MapArgs& a, int s, int64_t row, int held) {
  const int64_t entry = row >> a.page_shift;
  if (row < 0 || entry >= held) return -1;
  const int64_t page = a.table[static_cast<int64_t>(s) * a.width + entry];
  return (page << a.page_shift) + (row & ((int64_t{1} << a.page_shift) - 1));
}

// Inclusive sums over the block's threads of u and v, their totals behind; `part` holds sums for each wave.
__device__ __forceinline__ void block_scan(int& u, int& v, int (*part)[kTile / 64], int& u_all, int& v_all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u = wave_scan(u);
  v = wave_scan(v);
  __syncthreads();  // `part` of the call before is read
  if (lane == 63) {
    part[0][wave] = u;
    part[1][wave] = v;
  }
  __syncthreads();
  u_all = v_all = 0;
#pragma unroll
  for (int w = 0; w < kTile / 64; ++w) {
    if (w < wave) {
      u += part[0][w];
      v += part[1][w];
    }
    u_all += part[0][w];
    v_all += part[1][w];
  }
}

// The last of n ascending values that is <= x, the first being 0 or less.
__device__ __forceinline__ int last_up_to(const int* at, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (at[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Who finds the rows' slots: another launch; this block; further blocks, kTile rows at a time, which make the same sums for
// themselves and take what they need from what the first block leaves as it is: entries that are held, and the stack as it was.
enum { kSlotsLater, kSlotsHere, kSlotsByAll };

template <int SLOTS>
__global__ void __launch_bounds__(kTile) kv_page_map_kernel(MapArgs a) {
  constexpr int kRows = SLOTS == kSlotsLater ? 1 : kTile;
  __shared__ int part[2][kTile / 64];
  __shared__ int before[kTile], from[kTile];                       // pages taken before a sequence's, the entries they begin at
  __shared__ int backs[kTile], lows[kTile];                        // the same of pages that go back
  __shared__ int begin[kRows], holds[kRows];
  __shared__ int64_t first[kRows];
  const int tid = threadIdx.x;
  const bool moves = SLOTS != kSlotsByAll || blockIdx.x == 0;
  const int64_t there = within(a.count[0], 0, a.stack_size);
  const int tiles = (a.n_seq + kTile - 1) / kTile;
  MapSeq x = {};
  // back onto the stack
  int64_t top = there;
  int take = 0, taken_to = 0, takes = 0;  // of the tile: the sequence's pages to take, up to it, in all
  for (int t = 0; t < tiles; ++t) {
    const int s = t * kTile + tid;
    const bool live = s < a.n_seq;
    if (live) x = map_seq(a, s);
    const int back = live ? max(0, x.held - x.low) : 0;
    int total, sum = back;
    taken_to = take = live ? max(0, x.want - x.held) : 0;
    block_scan(sum, taken_to, part, total, takes);
    if (total == 0) continue;
    backs[tid] = sum - back;
    lows[tid] = x.low;
    __syncthreads();
    for (int i = tid; moves && i < total; i += kTile) {
      const int l = last_up_to(backs, min(kTile, a.n_seq - t * kTile), i);
      if (top + i < a.stack_size)
        a.stack[top + i] = a.table[static_cast<int64_t>(t * kTile + l) * a.width + lows[l] + (i - backs[l])];
    }
    top = min(top + total, a.stack_size);
    __syncthreads();
  }
  // and off it
  int64_t rank = 0, missing = 0;
  for (int t = 0; t < tiles; ++t) {
    const int s = t * kTile + tid;
    const bool live = s < a.n_seq;
    if (tiles > 1) {  // (else it is all there)
      if (live) x = map_seq(a, s);
      int none = 0, nothing;
      taken_to = take = live ? max(0, x.want - x.held) : 0;
      block_scan(none, taken_to, part, nothing, takes);
    }
    const int64_t mine = rank + taken_to - take;
    const int got = static_cast<int>(min(max(top - mine, int64_t{0}), static_cast<int64_t>(take)));
    const int now = take ? x.held + got : x.want;
    if (live) {
      missing += max(x.need - x.want, int64_t{0}) + (take - got);
      if (moves) a.held_out[s] = now;
    }
    before[tid] = taken_to - take;
    from[tid] = x.held;
    if constexpr (SLOTS != kSlotsLater) {
      begin[tid] = live ? static_cast<int>(x.begin) : 0x7FFFFFFF;
      first[tid] = x.pos;
      holds[tid] = now;
    }
    __syncthreads();
    for (int i = tid; moves && i < takes; i += kTile) {
      const int l = last_up_to(before, min(kTile, a.n_seq - t * kTile), i);
      if (rank + i < top)
        a.table[static_cast<int64_t>(t * kTile + l) * a.width + from[l] + (i - before[l])] = a.stack[top - 1 - rank - i];
    }
    if constexpr (SLOTS != kSlotsLater) {  // (one tile; of pages taken now not by the table: its entries may not be there yet)
      const unsigned end = static_cast<unsigned>(within(a.cu[a.n_seq], 0, a.rows));
      const auto taken = [&](int64_t place) -> int64_t {
        if (SLOTS == kSlotsHere || place < there) return a.stack[place];
        const int i = static_cast<int>(place - there), l = last_up_to(backs, a.n_seq, i);  // one that came back in this call
        return a.table[static_cast<int64_t>(l) * a.width + lows[l] + (i - backs[l])];
      };
      const unsigned step = SLOTS == kSlotsHere ? kTile : kTile * (gridDim.x - 1);  // (unsigned: past the end may be past 2^31)
      for (unsigned at_row = begin[0] + (SLOTS == kSlotsHere ? 0 : blockIdx.x - 1) * kTile + tid; at_row < end; at_row += step) {
        if (SLOTS == kSlotsByAll && moves) break;  // (it has enough to do)
        const int r = static_cast<int>(at_row), l = last_up_to(begin, a.n_seq, r);
        const int64_t at = first[l] + (r - begin[l]), entry = at >> a.page_shift;
        int64_t slot = -1;
        if (first[l] >= 0 && at >= 0 && entry < holds[l]) {
          const int64_t page = entry < from[l] ? a.table[static_cast<int64_t>(l) * a.width + entry]
                                               : taken(top - 1 - before[l] - (entry - from[l]));
          slot = (page << a.page_shift) + (at & ((int64_t{1} << a.page_shift) - 1));
        }
        a.slots[r] = slot;
      }
    }
    rank += takes;
    __syncthreads();
  }
  if (!moves) return;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) missing += __shfl_xor(missing, o);
  __shared__ int64_t lost[kTile / 64];
  if ((tid & 63) == 0) lost[tid / 64] = missing;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kTile / 64; ++w) missing += lost[w];
    a.count_out[0] = max(top - rank, int64_t{0});
    a.count_out[1] = missing;
  }
}

// A thread for each packed row, the tables done.
__global__ void __launch_bounds__(256) kv_page_slots_kernel(MapArgs a) {
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * 256 + (threadIdx.x & ~63), r = r0 + (threadIdx.x & 63);
  const auto start = [&](int s) { return within(a.cu[s], 0, a.rows); };
  int lo = last_started(a.n_seq, r0, start), hi = last_started(a.n_seq, r0 + 63, start) + 1;
  lo = max(lo, 0);
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (start(mid) <= r) lo = mid;
    else hi = mid;
  }
  const int64_t begin = start(lo);
  if (r < begin || r >= within(a.cu[lo + 1], begin, a.rows)) return;
  const int64_t pos = min(a.pos[lo], int64_t{1} << 62);
  a.slots[r] = pos < 0 ? -1 : map_slot(a, lo, pos + (r - begin), static_cast<int>(a.held_out[lo]));
}

// ------------------------------------------------------------------------------------------
// Append: a wave = 8 packed rows x 64 dims of a head (lane = row lane / 8, dims 8 (lane % 8)). K leaves as it came. Of V, 8 rows
// that fill one unit of 8 are turned in LDS and leave as 16 bytes a lane: they begin anywhere in the wave's 8 rows and end in the
// next wave's, so each wave looks at the slots of 8 rows before and after its own; other rows leave in pieces of 2 bytes.
// Bound by memory: 14300 rows of 8 heads of 128 (118 MB) 26.3 us, 4.5 TB/s; a token of each of 40 sequences 4.2 us, a launch.
// ------------------------------------------------------------------------------------------
struct AppendArgs {
  const uint16_t *k, *v;
  uint16_t *ck, *cv;
  int64_t k_row, k_head, v_row, v_head;
  const int64_t* slots;
  int64_t rows, n_slots;
  int heads, page_shift;
};

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

// Waits for this wave's LDS accesses; none moves across it.
__device__ __forceinline__ void lds_wave_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <int D>
__global__ void __launch_bounds__(256) kv_page_append_kernel(AppendArgs a) {
  __shared__ __align__(16) uint16_t turn[4][64][8];
  constexpr int kHalves = D / 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  const int parts = a.heads * kHalves;
  const int64_t r0 = unit / parts * 8;
  const int part = static_cast<int>(unit % parts), head = part / kHalves, d0 = part % kHalves * 64;
  if (r0 >= a.rows) return;  // no block barrier below
  // slots of rows r0 - 8 .. r0 + 15 in lanes 0 .. 23; -1 where there is none
  const int64_t at = r0 - 8 + lane;
  int64_t slot = -1;
  if (lane < 24 && at >= 0 && at < a.rows) slot = a.slots[at];
  if (slot < 0 || slot >= a.n_slots) slot = -1;
  // lane: whether its row and the 7 after it fill a unit
  const int64_t next = __shfl_down(slot, 1);
  const uint64_t follows = __builtin_amdgcn_ballot_w64(slot >= 0 && next == slot + 1);
  const uint64_t starts = __builtin_amdgcn_ballot_w64(slot >= 0 && (slot & 7) == 0);
  uint64_t run = follows & (follows >> 1);
  run &= run >> 2;                                              // 4 in a row
  run &= (run >> 3);                                            // 7 in a row
  const uint64_t whole = starts & run & 0xFFFF;                 // rows r0 - 8 .. r0 + 7 that begin a whole unit
  uint64_t covered = 0;                                         // of rows r0 .. r0 + 7, by a whole unit (at most two reach them)
  for (uint64_t w = whole; w; w &= w - 1) covered |= uint64_t{0xFF} << __builtin_ctzll(w);
  const int r = lane >> 3, d = d0 + 8 * (lane & 7);
  const int64_t page_rows = int64_t{1} << a.page_shift, low = page_rows - 1;
  // the head's rows of a slot's page begin at this row of the cache
  const auto base = [&](int64_t s) { return ((s >> a.page_shift) * a.heads + head) << a.page_shift; };
  const int64_t mine = __shfl(slot, 8 + r);
  u16x8 kx = {}, vx = {};
  if (mine >= 0) {
    kx = *reinterpret_cast<const u16x8*>(a.k + (r0 + r) * a.k_row + head * a.k_head + d);
    vx = *reinterpret_cast<const u16x8*>(a.v + (r0 + r) * a.v_row + head * a.v_head + d);
  }
  const int begins = (whole >> 8) ? __builtin_ctzll(whole >> 8) : -1;  // own row that begins a whole unit, at most one
  u16x8 ux = vx;
  if (begins > 0) ux = *reinterpret_cast<const u16x8*>(a.v + (r0 + begins + r) * a.v_row + head * a.v_head + d);
  if (mine >= 0) {
    *reinterpret_cast<u16x8*>(a.ck + (base(mine) + (mine & low)) * D + d) = kx;
    if (!((covered >> (8 + r)) & 1)) {
      uint16_t* to = a.cv + (base(mine) + (mine & low & ~int64_t{7})) * D + static_cast<int64_t>(d) * 8 + (mine & 7);
#pragma unroll
      for (int e = 0; e < 8; ++e) to[8 * e] = vx[e];
    }
  }
  if (begins >= 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) turn[wave][8 * (lane & 7) + e][r] = ux[e];
    lds_wave_done();
    const int64_t s = __shfl(slot, 8 + begins);
    *reinterpret_cast<u16x8*>(a.cv + (base(s) + (s & low)) * D + static_cast<int64_t>(d0 + lane) * 8) =
        *reinterpret_cast<const u16x8*>(turn[wave][lane]);
  }
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool rows_ok(const void* p, int64_t row, int64_t head) { return aligned(p, 16) && row % 8 == 0 && head % 8 == 0; }

// Slots that one block finds beside the map (us in one launch / two: 64 sequences with 1500 rows 6.2 / 8.1, with 3400 7.5 / 8.1,
// 8 with 6300 8.1 / 7.2).
constexpr int64_t kOneBlockRows = 4 * kTile, kMostBlocks = 512;

}  // namespace
}  // namespace fw

using namespace fw;

extern "C" int fw_kv_page_map(const int64_t* pos, const int64_t* cu, int32_t* table, const int64_t* held, const int64_t* own,
                              int32_t* stack, const int64_t* count, int64_t* held_out, int64_t* count_out, int64_t* slots,
                              int n_seq, int width, int64_t stack_size, int64_t rows, int page, hipStream_t stream) {
  const int shift = page_shift_of(page);
  if (shift < 0) return fw_fail(FW_EINVAL, "kv_page_map: page must be 16, 32, 64, 128 or 256 rows");
  if (n_seq <= 0 || width <= 0 || stack_size < 0 || rows < 0)
    return fw_fail(FW_EINVAL, "kv_page_map: n_seq and width must be positive, sizes not negative");
  // entries of kTile sequences are counted in 32 bits, as are packed rows
  if (width > (1 << 20) || rows > 0x7FFFFF00) return fw_fail(FW_EINVAL, "kv_page_map: at most 2^20 pages a sequence and 2^31 - 256 rows");
  if (!pos || !cu || !table || !held || !count || !held_out || !count_out || (stack_size > 0 && !stack) || (rows > 0 && !slots))
    return fw_fail(FW_EINVAL, "kv_page_map: null pointer");
  const MapArgs a{pos, cu, held, own, count, table, stack, held_out, count_out, slots, rows, stack_size, n_seq, width, shift};
  // what the first block writes while others read: only with outputs of their own there is nothing of the inputs among it
  const auto apart = [&](const int64_t* out, int64_t n) {
    const auto from = [&](const int64_t* in, int64_t m) { return !in || out + n <= in || in + m <= out; };
    return from(pos, n_seq) && from(cu, n_seq + 1) && from(held, n_seq) && from(own, n_seq) && from(count, 2);
  };
  const bool by_all = n_seq <= kTile && rows > 0 && apart(held_out, n_seq) && apart(count_out, 2);
  const bool one = n_seq <= kTile && rows <= kOneBlockRows;
  const int64_t blocks = std::min<int64_t>((rows + kTile - 1) / kTile, kMostBlocks);
  if (by_all) hipLaunchKernelGGL(kv_page_map_kernel<kSlotsByAll>, dim3(static_cast<unsigned>(blocks) + 1), dim3(kTile), 0, stream, a);
  else if (one) hipLaunchKernelGGL(kv_page_map_kernel<kSlotsHere>, dim3(1), dim3(kTile), 0, stream, a);
  else hipLaunchKernelGGL(kv_page_map_kernel<kSlotsLater>, dim3(1), dim3(kTile), 0, stream, a);
  if (const int rc = fw_check_launch("kv_page_map")) return rc;
  if (by_all || one || rows == 0) return FW_OK;
  hipLaunchKernelGGL(kv_page_slots_kernel, dim3(static_cast<unsigned>((rows + 255) / 256)), dim3(256), 0, stream, a);
  return fw_check_launch("kv_page_map slots");
}

extern "C" int fw_kv_page_append(const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                                 const int64_t* slots, int64_t rows, void* k_pages, void* v_pages, int n_pages, int kv_heads,
                                 int page, int head_dim, hipStream_t stream) {
  const int shift = page_shift_of(page);
  if (shift < 0) return fw_fail(FW_EINVAL, "kv_page_append: page must be 16, 32, 64, 128 or 256 rows");
  if (head_dim != 64 && head_dim != 128) return fw_fail(FW_EINVAL, "kv_page_append: head_dim must be 64 or 128");
  if (n_pages <= 0 || kv_heads <= 0 || rows < 0)
    return fw_fail(FW_EINVAL, "kv_page_append: n_pages and kv_heads must be positive, rows not negative");
  if (!k_pages || !v_pages || (rows > 0 && (!k || !v || !slots))) return fw_fail(FW_EINVAL, "kv_page_append: null pointer");
  if (!aligned(k_pages, 16) || !aligned(v_pages, 16) || (rows > 0 && (!rows_ok(k, k_row, k_head) || !rows_ok(v, v_row, v_head))))
    return fw_fail(FW_EINVAL, "kv_page_append: rows and pages must be 16-byte aligned, strides multiples of 8");
  const int64_t parts = static_cast<int64_t>(kv_heads) * (head_dim / 64);
  if ((rows + 7) / 8 > 0xFFFFFFFFll / 256 * 4 / parts) return fw_fail(FW_EINVAL, "kv_page_append: too many rows");
  if (rows == 0) return FW_OK;
  const AppendArgs a{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), static_cast<uint16_t*>(k_pages),
                     static_cast<uint16_t*>(v_pages), k_row, k_head, v_row, v_head, slots, rows,
                     static_cast<int64_t>(n_pages) << shift, kv_heads, shift};
  const unsigned blocks = static_cast<unsigned>(((rows + 7) / 8 * parts + 3) / 4);
  if (head_dim == 64) hipLaunchKernelGGL(kv_page_append_kernel<64>, dim3(blocks), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(kv_page_append_kernel<128>, dim3(blocks), dim3(256), 0, stream, a);
  return fw_check_launch("kv_page_append");
}
