// A key/value cache in pages. Layout (P = 2^page_shift rows a page, D = 64 or 128, 16-bit values):
//   k [page][head][P][D]          row-major: a lane's dims of a Q K product in one load
//   v [page][head][P / 8][D][8]   8 rows of a dim in 16 bytes: a lane's keys of a P V product in one load
// Slot x is row x % P of page x / P; a negative one is no place. Row j of sequence s lies in page table[s][j / P].
#pragma once

namespace fw {

// log2 of a page's rows, or -1 for a size that pages do not have: 16 to 256 rows.
inline int page_shift_of(int page) {
  for (int s = 4; s <= 8; ++s)
    if (page == 1 << s) return s;
  return -1;
}

}  // namespace fw
