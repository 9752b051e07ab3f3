// error_bits.h -- the bits of a backend's error word, which its kernels set
// and sam3b200_backend_synchronize reads and clears.
#pragma once

namespace b200 {

// Bits that say what was wrong with a call's data.  Every other bit is a
// bounded wait that ran out; the kernels choose theirs as they like (each
// pipeline kernel asserts that it keeps out of kErrData).
constexpr int kErrData = 0x00ff0000;
constexpr int kErrGetRowsIndex = 1 << 20;  // get_rows: an index outside [0, nrows)
constexpr int kErrKvPage = 1 << 21;        // a block table names a page outside [0, n_pages)
constexpr int kErrKvBatch = 1 << 22;       // row_start / kv_len contradict the batch's sizes
static_assert(((kErrGetRowsIndex | kErrKvPage | kErrKvBatch) & ~kErrData) == 0, "errors of data");

}  // namespace b200
