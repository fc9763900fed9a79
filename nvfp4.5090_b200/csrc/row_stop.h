// Leaving a loop over rows when a bounded wait ran out.
//
// Every row has one barrier of the CTA, and the threads must leave the loop at
// the same row: some at a later barrier than others would wait for one another
// without a limit.  So a thread whose wait ran out lowers a shared number to
// the row at whose barrier all are to leave, and every thread compares it with
// its row right behind that row's barrier.  A wait before the barrier of row i
// stops the loop there.  A wait after it stops it at the next row's: until
// that barrier the number can only become i + 1, so whether a thread reads it
// before or after, it goes on with row i.
#pragma once

#ifdef __CUDACC__
#define ROW_STOP_FN __host__ __device__ __forceinline__
#else
#define ROW_STOP_FN inline
#endif

namespace nvfp4b200 {
namespace row_stop {

constexpr int NEVER = 0x7FFFFFFF;   // the shared number at first

ROW_STOP_FN int before_barrier(int row) { return row; }
ROW_STOP_FN int after_barrier(int row) { return row + 1; }
// Right behind the barrier of `row`, before anything that the row still does.
ROW_STOP_FN bool leaves(int stop, int row) { return stop <= row; }

}  // namespace row_stop
}  // namespace nvfp4b200
