// Which tile counter a launch of the GEMM takes.  Host code, no CUDA.
//
// Two launches that run at the same time must not claim tiles from one
// counter.  Launches of one stream run one after another, so a stream keeps one
// counter for good.  A launch that is captured into a graph runs whenever the
// graph does, on any stream: it has a counter to itself until the graph and
// all that was instantiated from it are gone.  A launch that finds no counter
// free gets -1 and walks its tiles in a fixed order.
#pragma once

#include <cstdint>
#include <mutex>

namespace nvfp4b200 {

// Plain arrays: nothing here allocates, so nothing throws through a C entry point.
template <int STREAMS, int GRAPHS>
class SchedSlots {   // of one device
 public:
  static constexpr int COUNT = STREAMS + GRAPHS;

  // The counter of a stream, by an id that no other stream ever has.
  int of_stream(uint64_t id) {
    std::lock_guard<std::mutex> lock(mu_);
    for (int i = 0; i < streams_; ++i)
      if (ids_[i] == id) return i;
    if (streams_ == STREAMS) return -1;
    ids_[streams_] = id;
    return streams_++;
  }

  // A counter for one captured launch, until give_back.
  int take() {
    std::lock_guard<std::mutex> lock(mu_);
    if (fresh_ < GRAPHS) return STREAMS + fresh_++;
    if (waiting_ == 0) return -1;
    const int slot = back_[first_];   // the one that has been back the longest
    first_ = (first_ + 1) % GRAPHS;
    --waiting_;
    return slot;
  }

  void give_back(int slot) {   // one that take() gave: at most GRAPHS are out
    std::lock_guard<std::mutex> lock(mu_);
    back_[(first_ + waiting_++) % GRAPHS] = slot;
  }

 private:
  std::mutex mu_;
  uint64_t ids_[STREAMS] = {};
  int streams_ = 0, fresh_ = 0;
  int back_[GRAPHS] = {};   // given back: waiting_ of them from first_ on, around the end
  int first_ = 0, waiting_ = 0;
};

}  // namespace nvfp4b200
