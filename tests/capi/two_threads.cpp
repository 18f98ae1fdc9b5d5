// Two contexts, each called from a thread of its own as fast as it goes, on
// rows of different length: the number of calls that were refused.
#include <atomic>
#include <thread>

#include "heliox_b200.h"

extern "C" int two_threads(hx_ctx* const* ctx, const hx_readout* rows, int k, int32_t* const* idx, void* const* val, int calls) {
    std::atomic<int> refused{0}, ready{0};
    const auto work = [&](int j) {
        ready++;
        while (ready < 2) std::this_thread::yield();
        for (int n = 0; n < calls; n++) refused += hx_top_logits_dev(ctx[j], &rows[j], k, 1.0, idx[j], val[j], nullptr) != 0;
    };
    std::thread a(work, 0), b(work, 1);
    a.join();
    b.join();
    return refused;
}
