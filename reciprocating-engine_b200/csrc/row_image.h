// How a row of any alignment is copied to shared memory: its image keeps the
// bytes between the row's 16-byte boundary and its first element (the lead) as
// a gap, so that both sides of every copy are aligned alike, and each copy
// reads bytes of the row alone.  Copies are of 16 bytes (the last of fewer:
// the rest of its destination is zero-filled), of 4 in front of the first
// whole piece, and there is no copy of a 16-bit element that begins a row in
// the middle of 4 bytes: row_odd says that there is one, which takes a load
// and a store.
// tests/test_fp8_blocks_calls.py checks on the CPU that the accesses are
// aligned and cover the row exactly, for every alignment.
#pragma once
#include <stdint.h>

#ifndef RENG_HD
#ifdef __CUDACC__
#define RENG_HD __host__ __device__ __forceinline__
#else
#define RENG_HD inline
#endif
#endif

namespace reng {

RENG_HD int row_lead(const void* row) { return (int)((uintptr_t)row & 15); }

// The row's first element is not copied by row_word.
RENG_HD bool row_odd(int lead) { return (lead & 3) != 0; }

// Word w of the image's first 16 bytes (w 0 to 3): copy(offset, size), offsets
// from the row's 16-byte boundary (source) and from the image's start
// (destination) alike, size at most 4.
template <typename Copy>
RENG_HD void row_word(int lead, int bytes, int w, Copy copy) {
    const int at = 4 * w, left = lead + bytes - at;
    if (at >= lead && left > 0) copy(at, left < 4 ? left : 4);
}

// Offsets from 16 to row_whole: whole pieces of 16.
RENG_HD int row_whole(int lead, int bytes) { return (lead + bytes) & ~15; }

// The row's last piece, from there on: copy(offset, size), size below 16.
template <typename Copy>
RENG_HD void row_rest(int lead, int bytes, Copy copy) {
    const int at = row_whole(lead, bytes), left = lead + bytes - at;
    if (at >= 16 && left > 0) copy(at, left);
}

}  // namespace reng
