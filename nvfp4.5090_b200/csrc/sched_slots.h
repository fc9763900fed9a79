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
#include <deque>
#include <mutex>
#include <unordered_map>

namespace nvfp4b200 {

template <int STREAMS, int GRAPHS>
class SchedSlots {   // of one device
 public:
  static constexpr int COUNT = STREAMS + GRAPHS;

  // The counter of a stream, by an id that no other stream ever has.
  int of_stream(uint64_t id) {
    std::lock_guard<std::mutex> lock(mu_);
    const auto at = streams_.find(id);
    if (at != streams_.end()) return at->second;
    if ((int)streams_.size() == STREAMS) return -1;
    const int slot = (int)streams_.size();
    streams_.emplace(id, slot);
    return slot;
  }

  // A counter for one captured launch, until give_back.
  int take() {
    std::lock_guard<std::mutex> lock(mu_);
    if (fresh_ < GRAPHS) return STREAMS + fresh_++;
    if (back_.empty()) return -1;
    const int slot = back_.front();   // the one that has been back the longest
    back_.pop_front();
    return slot;
  }

  void give_back(int slot) {
    std::lock_guard<std::mutex> lock(mu_);
    back_.push_back(slot);
  }

 private:
  std::mutex mu_;
  std::unordered_map<uint64_t, int> streams_;
  std::deque<int> back_;
  int fresh_ = 0;
};

}  // namespace nvfp4b200
