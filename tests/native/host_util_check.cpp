// Host-only checks of kd_host.h.  Prints "OK" or the first failure.  Built and run by tests/test_fp8_edges_cpu.py.
#include <cstdio>
#include <cstdlib>
#include <set>

#include "kd_host.h"

// rows_overlap against every pair of rows, over all small strides and counts.
static int check_rows_overlap() {
    for (uint64_t bytes = 1; bytes <= 4; ++bytes)
        for (uint64_t nb1 = 0; nb1 <= 14; ++nb1)
            for (uint64_t nb2 = 0; nb2 <= 14; ++nb2)
                for (int64_t L = 0; L <= 5; ++L)
                    for (int64_t N = 0; N <= 5; ++N) {
                        std::set<uint64_t> used;
                        bool want = false;
                        for (int64_t l = 0; l < L; ++l)
                            for (int64_t n = 0; n < N; ++n)
                                for (uint64_t b = 0; b < bytes; ++b) want |= !used.insert(l * nb1 + n * nb2 + b).second;
                        if (kd::rows_overlap(bytes, nb1, nb2, L, N) != want) {
                            printf("rows_overlap(%llu, %llu, %llu, %lld, %lld) is not %d\n", (unsigned long long)bytes,
                                   (unsigned long long)nb1, (unsigned long long)nb2, (long long)L, (long long)N, want);
                            return 1;
                        }
                    }
    // the largest counts and strides: no overflow, and no long loop
    const uint64_t big = 1ull << 62;
    if (kd::rows_overlap(64, 64, 1ull << 40, 1 << 12, 1 << 12) || !kd::rows_overlap(64, 65, 64, 1 << 12, 1 << 12) ||
        kd::rows_overlap(64, big, 64, 1 << 12, 1 << 12) || !kd::rows_overlap(64, big, big + 63, 1 << 12, 1 << 12)) {
        printf("rows_overlap: large sizes\n");
        return 1;
    }
    return 0;
}

// PerDevice: failures are asked again, answers are kept, each for its own device; devices beyond the table are asked anew.
static int check_per_device() {
    kd::PerDevice v;
    int asked = 0;
    auto answer = [&](int n) { return [&asked, n] { return ++asked, n; }; };
    const bool good = v.get(0, answer(0)) == 0 && v.get(0, answer(-3)) == -3 && v.get(0, answer(74)) == 74 && asked == 3 &&
                      v.get(0, answer(5)) == 74 && asked == 3 && v.get(1, answer(66)) == 66 && v.get(0, answer(1)) == 74 &&
                      v.get(1, answer(1)) == 66 && asked == 4 && v.get(64, answer(7)) == 7 && v.get(64, answer(8)) == 8 &&
                      v.get(-1, answer(9)) == 9 && asked == 7;
    if (!good) printf("PerDevice\n");
    return good ? 0 : 1;
}

int main() {
    const int bad = check_rows_overlap() + check_per_device();
    if (!bad) printf("OK\n");
    return bad;
}
