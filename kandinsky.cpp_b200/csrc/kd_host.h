// kd_host.h -- host-side helpers of the library that need no CUDA.
#pragma once

#include <atomic>
#include <cstdint>

namespace kd {

// A positive number for each device, asked for on first use there and kept.  What is not positive (a question that
// failed) is given back and not kept, so that the next call asks again.  Threads may ask at the same time.
class PerDevice {
public:
    template <typename Ask>
    int get(int device, Ask&& ask) {
        const bool room = device >= 0 && device < kDevices;
        if (room) {
            const int v = known_[device].load(std::memory_order_acquire);
            if (v > 0) return v;
        }
        const int v = ask();
        if (room && v > 0) known_[device].store(v, std::memory_order_release);
        return v;
    }

private:
    static constexpr int kDevices = 64;
    std::atomic<int> known_[kDevices] = {};
};

// Whether rows of `bytes` > 0 that start at l * nb1 + n * nb2 (0 <= l < L, 0 <= n < N) share a byte.
inline bool rows_overlap(uint64_t bytes, uint64_t nb1, uint64_t nb2, int64_t L, int64_t N) {
    if (L <= 0 || N <= 0) return false;
    if ((L > 1 && nb1 < bytes) || (N > 1 && nb2 < bytes)) return true;
    if (L == 1 || N == 1) return false;
    using Wide = unsigned __int128;
    const bool swap = nb1 > nb2;
    const Wide step = swap ? nb2 : nb1, far = swap ? nb1 : nb2;  // bytes <= step <= far
    const Wide count = (Wide)(swap ? N : L), groups = (Wide)(swap ? L : N);
    if (step * (count - 1) + bytes <= far) return false;  // a group of rows ends before the next starts, as in most views
    // i steps of `far` against the j steps of `step` below them, and the j + 1 above; from j = count on they lie at
    // least a step, so a row, past all rows of the first group
    for (Wide i = 1; i < groups; ++i) {
        const Wide j = i * far / step, rest = i * far % step;
        if (j >= count) break;
        if (rest < bytes || (j + 1 < count && step - rest < bytes)) return true;
    }
    return false;
}

}  // namespace kd
