// ceil_div of af_common.h: launches are sized with it from bounds that callers may set as high as INT32_MAX.
#include <cstdint>
#include <cstdio>

#include "af_common.h"

int main() {
    int bad = 0;
    for (int b : {1, 2, 3, 32, 51, 255, 256, 512, 1 << 20, INT32_MAX})
        for (int64_t near : {int64_t(0), int64_t(b), int64_t(7) * b, int64_t(1) << 30, int64_t(INT32_MAX) - 300,
                             int64_t(INT32_MAX)})
            for (int64_t a = near - 600; a <= near + 600; ++a) {
                if (a < 0 || a > INT32_MAX) continue;
                const int64_t want = (a + b - 1) / b;
                if (af::ceil_div(int(a), b) != want && bad++ < 5)
                    std::printf("ceil_div(%lld, %d) is %d\n", (long long)a, b, af::ceil_div(int(a), b));
            }
    if (bad) return 1;
    std::printf("ok\n");
    return 0;
}
