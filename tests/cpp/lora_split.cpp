// How the adapters' first product cuts K (af_lora_split.h), for every k: no part is empty, parts abut and cover K,
// and every load of the form that goes through LDS lies within its row, each element of K in one of them.
#include <cstdio>
#include <vector>

#include "af_lora_split.h"

static int fail(const char* what, int k, int splits, int split) {
    std::printf("%s: k %d, %d splits, split %d\n", what, k, splits, split);
    return 1;
}

static int check(int k) {
    const af::LoraSplit s = af::lora_split(k);
    if (s.parts < 1 || s.parts > af::kLoraParts || s.part_k % 256) return fail("split", k, s.parts, 0);
    for (int splits : {1, s.parts}) {
        int end = 0;
        std::vector<char> seen(size_t(k) / 8, 0);
        for (int split = 0; split < splits; ++split) {
            const af::LoraRange r = af::lora_range(k, s.part_k, splits, split);
            if (r.k0 != end || r.k1 <= r.k0 || r.k1 > k) return fail("part", k, splits, split);
            end = r.k1;
            // the kernel's count: two pieces ahead, then one for each that is used
            int ahead = r.pieces, issued = 0;
            for (int call = 0; call < 2 + r.pieces; ++call) {
                if (ahead == 0) continue;
                --ahead;
                for (int eighth = 0; eighth < 8; ++eighth) {
                    int at = r.k0 + af::kLoraPiece * issued + 8 * eighth;
                    if (ahead == 0) at += af::lora_pull_back(k, r, eighth);
                    if (at < 0 || at + 8 > k || at % 8) return fail("load outside the row", k, splits, split);
                    seen[size_t(at) / 8] = 1;
                }
                ++issued;
            }
            if (issued != r.pieces || ahead != 0) return fail("loads", k, splits, split);
        }
        if (end != k) return fail("end", k, splits, splits);
        for (char c : seen)
            if (!c) return fail("not read", k, splits, 0);
    }
    return 0;
}

int main() {
    int bad = 0;
    for (int k = 8; k <= 32768; k += 8) bad += check(k);
    for (int k = 40000; k <= 1 << 24; k += 8 * 98765) bad += check(k);
    bad += check(1 << 24);
    if (bad) return 1;
    std::printf("ok\n");
    return 0;
}
