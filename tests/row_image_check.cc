// CPU check of a row's copy to its image in shared memory
// (reciprocating-engine_b200/csrc/row_image.h): for rows of 2- and 4-byte
// elements at every alignment and of many lengths, every access is aligned to
// its size, none leaves the row, and each byte of the row is copied once.
#include <cstdio>
#include <vector>

#include "row_image.h"

int main() {
    long long bad = 0, cases = 0;
    for (int esize : {2, 4})
        for (int lead = 0; lead < 16; lead += esize)
            for (int n = 1; n <= 300; n++) {
                cases++;
                const int bytes = n * esize, end = lead + bytes, image = (bytes + 15) / 16 * 16 + 16;
                std::vector<int> seen(end, 0);
                if (reng::row_lead((const void*)(uintptr_t)(4096 + lead)) != lead) bad++;
                auto copy = [&](int o, int size, int n) {
                    if (o % n || size < 1 || size > n || o < lead || o + size > end || o + n > image) bad++;
                    for (int b = o; b < o + size && b < end; b++) seen[b]++;
                };
                for (int w = 0; w < 4; w++) reng::row_word(lead, bytes, w, [&](int o, int size) { copy(o, size, 4); });
                for (int at = 16; at < reng::row_whole(lead, bytes); at += 16) copy(at, 16, 16);
                reng::row_rest(lead, bytes, [&](int o, int size) { copy(o, size, 16); });
                if (reng::row_odd(lead)) {
                    if (esize != 2 || lead % 2) bad++;
                    seen[lead]++, seen[lead + 1]++;
                }
                for (int b = 0; b < end; b++)
                    if (seen[b] != (b >= lead)) bad++;
            }
    printf("cases %lld bad %lld\n", cases, bad);
    return bad ? 1 : 0;
}
