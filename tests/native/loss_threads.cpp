// Threads that call cugo_b200_policy_loss at the same time, without an interpreter between
// them: thread k takes rows of vocab[k] entries on stream[k].
#include <atomic>
#include <cstdint>
#include <thread>
#include <vector>

#include "../../include/cugo_b200.h"

extern "C" __attribute__((visibility("default"))) int64_t loss_threads(
    decltype(&cugo_b200_policy_loss) call, int threads, int calls, int64_t rows, const int64_t* vocab,
    void* const* logits, void* const* dlogits, void* const* scratch, int64_t scratch_bytes, cudaStream_t const* stream,
    const int64_t* actions, const float* zeros) {
  std::atomic<int64_t> ready{0}, failed{0};
  std::vector<std::thread> all;
  for (int k = 0; k < threads; ++k)
    all.emplace_back([&, k] {
      ++ready;
      while (ready < threads) std::this_thread::yield();
      for (int i = 0; i < calls; ++i)
        if (call(logits[k], vocab[k], 1, nullptr, 0, nullptr, 0, actions, zeros, zeros, nullptr, nullptr, rows,
                 vocab[k], 0.2f, 0.2f, 0.0f, 0.0f, nullptr, nullptr, 0.0f, nullptr, 1.0f, nullptr, dlogits[k],
                 vocab[k], 1, vocab[k], nullptr, nullptr, nullptr, scratch[k], scratch_bytes, stream[k]))
          ++failed;
    });
  for (std::thread& t : all) t.join();
  return failed;
}
