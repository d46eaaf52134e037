// Slices of rows by the widest of their arrays (score_slices.h): never empty, never more than the rows or than 256 MB of 32-bit numbers but for a single
// row, and not smaller than they have to be.
#include <cstdio>
#include <initializer_list>

#include "../../thundergbm_amd/csrc/score_slices.h"

#define CHECK(c) \
    if (!(c)) { std::printf("line %d: %s (%lld rows of %lld: %lld)\n", __LINE__, #c, rows, widest, most); return 1; }

int main() {
    const long long room = 1ll << 28;
    for (long long rows : {1ll, 2ll, 1000ll, 1024ll, 1025ll, 6700000ll, (1ll << 31) - 1})
        for (long long widest : {1ll, 3ll, 257ll, 4096ll, 65536ll, 1ll << 22, 1ll << 26, (1ll << 26) + 1, 1ll << 40}) {
            const long long most = tgbm::rows_of_a_slice(rows, widest);
            CHECK(most >= 1 && most <= rows);
            CHECK(most == 1 || 4 * most * widest <= room);
            CHECK(most == rows || 4 * (most + 1) * widest > room);
        }
    std::printf("ok\n");
    return 0;
}
