// CPU check of how lists of tensors and long states are dealt out to launches
// (jax-gs_amd/csrc/gs_pieces.h), built and run by tests/test_step_pieces.py: every workgroup of every
// tensor with a gradient once and in order, no launch of 2^32 work items or of too many records.
//
// Output (one line): lists, launches, most workgroups of a launch, faults
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "gs_pieces.h"

int main(int argc, char** argv) {
  const long lists = argc > 1 ? atol(argv[1]) : 1000;
  std::mt19937_64 rng(argc > 2 ? strtoull(argv[2], nullptr, 10) : 1ull);
  std::uniform_real_distribution<double> u(0.0, 1.0);
  const int64_t most_count = ((int64_t)1 << 40) - 256;
  long faults = 0, launches_seen = 0;
  int64_t most = 0;
  for (long s = 0; s < lists; ++s) {
    const int n = (int)(rng() % (s % 7 == 0 ? 4 : 300));
    // small lists, lists with some tensor beyond one launch, and lists whose sum is
    const double top = s % 3 == 0 ? 20.0 : s % 3 == 1 ? 34.0 : 40.0;
    std::vector<int64_t> counts(n);
    std::vector<const void*> grads(n);
    for (int i = 0; i < n; ++i) {
      counts[i] = rng() % 9 == 0 ? 0 : std::min(most_count, (int64_t)std::exp2(u(rng) * top));
      if (rng() % 16 == 0) counts[i] = std::min(most_count, (counts[i] >> 30 << 30) + (int64_t)(rng() % 3) - 1);
      if (counts[i] < 0) counts[i] = 0;
      grads[i] = rng() % 8 == 0 ? nullptr : &counts;
    }
    if (n && s % 50 == 1) counts[n / 2] = most_count;
    gs::StepPieces pieces(n, grads.data(), counts.data());
    int tensor = -1;
    int64_t at = 0, launches = 0, records = 0;  // workgroups of `tensor` seen
    auto close = [&](int to) {                  // the tensor before is whole, and those between take no part
      if (tensor >= 0) faults += at != (counts[tensor] + gs::kStepChunk - 1) / gs::kStepChunk;
      for (int i = tensor + 1; i < to; ++i) faults += grads[i] && counts[i] > 0;
      at = 0;
      tensor = to;
    };
    while (!pieces.done()) {
      gs::StepPiece out[gs::kStepTensors];
      int64_t groups = 0;
      const int k = pieces.next(out, groups);
      ++launches;
      records += k;
      if (k < 1 || k > gs::kStepTensors || groups < 1 || groups * 256 >= (int64_t)1 << 32) {
        ++faults;
        break;
      }
      most = std::max(most, groups);
      for (int j = 0; j < k; ++j) {
        const int64_t length = (j + 1 < k ? out[j + 1].begin : groups) - out[j].begin;
        if (out[j].tensor != tensor) close(out[j].tensor);
        faults += out[j].tensor >= n || !grads[out[j].tensor] || length < 1 || (j == 0 && out[j].begin != 0);
        faults += out[j].piece < 0 || out[j].piece > 0xffff || out[j].piece * gs::kPieceGroups != at;
        at += length;
      }
    }
    close(n);
    // lists of what fits one launch many times over: as few launches as the records need
    if (s % 3 == 0 && s % 50 != 1) faults += launches != (records + gs::kStepTensors - 1) / gs::kStepTensors;
    launches_seen += launches;

    // conversions
    const int64_t blocks = std::min(most_count, (int64_t)std::exp2(u(rng) * 40.0)) / 256;
    int64_t first = 0;
    while (first < blocks) {
      const int64_t here = gs::conversion_blocks(first, blocks);
      faults += here < 1 || (here + 3) / 4 * 256 >= (int64_t)1 << 32;
      first += here;
    }
    faults += first != blocks;
  }
  std::printf("%ld %ld %lld %ld\n", lists, launches_seen, (long long)most, faults);
  return faults == 0 ? 0 : 1;
}
