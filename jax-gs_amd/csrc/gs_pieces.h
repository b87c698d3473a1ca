// How lists of tensors and long arrays are dealt out to launches, on the host.
#pragma once

#include <algorithm>
#include <cstdint>

namespace gs {

// Workgroups of 256 in one launch: HIP takes fewer than 2^32 work items in a dimension.
constexpr int64_t kMaxGroups = ((int64_t)1 << 24) - 1;

constexpr int kStepTensors = 76;  // records per launch of the step: its argument block stays below 4 KiB
constexpr int kStepChunk = 1024;  // elements per workgroup

// A tensor of more workgroups than this is several records, so that any tensor fits some launch:
// 2^30 elements each, at most 2^10 of them.
constexpr int64_t kPieceGroups = (int64_t)1 << 20;

struct StepPiece {
  int tensor;
  int piece;       // from workgroup piece * kPieceGroups of the tensor on
  int64_t begin;   // its first workgroup in the launch
};

// Deals the tensors that have a gradient and elements out to launches, in order.
struct StepPieces {
  int num;
  const void* const* grads;
  const int64_t* counts;
  int tensor = 0, piece = 0;  // next
  int each;                   // records per launch, split evenly

  StepPieces(int num_, const void* const* grads_, const int64_t* counts_) : num(num_), grads(grads_), counts(counts_) {
    int64_t some = 0;
    for (int i = 0; i < num; ++i)
      if (grads[i]) some += (groups_of(i) + kPieceGroups - 1) / kPieceGroups;
    const int64_t launches = (some + kStepTensors - 1) / kStepTensors;
    each = launches > 0 ? (int)((some + launches - 1) / launches) : 0;
    skip();
  }
  int64_t groups_of(int i) const { return (counts[i] + kStepChunk - 1) / kStepChunk; }
  void skip() {
    while (tensor < num && (!grads[tensor] || counts[tensor] == 0)) ++tensor;
  }
  bool done() const { return tensor >= num; }
  // The records of the next launch and its workgroups; returns how many records (none only when done).
  int next(StepPiece (&out)[kStepTensors], int64_t& groups) {
    int k = 0;
    groups = 0;
    while (!done() && k < each) {
      const int64_t from = piece * kPieceGroups, all = groups_of(tensor), more = std::min(all - from, kPieceGroups);
      if (groups + more > kMaxGroups) break;
      out[k++] = StepPiece{tensor, piece, groups};
      groups += more;
      if (from + more < all) {
        ++piece;
      } else {
        piece = 0;
        ++tensor;
        skip();
      }
    }
    return k;
  }
};

// A conversion takes four blocks a workgroup: how many of the blocks from `first` on go into one launch.
inline int64_t conversion_blocks(int64_t first, int64_t blocks) { return std::min(blocks - first, kMaxGroups * 4); }

}  // namespace gs
