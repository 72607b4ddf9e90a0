// Walks random items through the rings of the two-halved attention kernel and checks that no half waits for a fill of a values' slot
// that it may take for another: a wait by parity tells only neighbouring fills apart, so before it waits for block n of a ring of R
// slots, block n - R has to have landed as far as the half can know.
//
// What it can know: the issuing warp walks the blocks of all items in order; ahead of a half's product with block n it waits for the
// values of block n, ahead of the scores of block n it has issued that half's product with the block before (where the item
// has one), and an item's first scores come behind all products of the item before.  A half learns of it by the scores and the
// last product of its own blocks.  Prints "ok" and the number of waits that followed blocks the half sat out.
#include <algorithm>
#include <cstdio>
#include <random>

#include "../eptq_b200/csrc/attention_schedule.cuh"

using namespace eptq;

static std::mt19937 generator(2);
static int from(int a, int b) { return a + static_cast<int>(generator() % static_cast<unsigned>(b - a + 1)); }

int main() {
    long behind = 0;
    for (int walk = 0; walk < 20000; ++walk) {
        const int ring = from(0, 1) ? 2 : 5, kb = 128, per_half = from(0, 1) ? 32 : from(1, 128);
        const bool short_items = from(0, 1);
        long long base = 0;                    // blocks of the items before
        long long known[2] = {-1, -1};         // the last block whose values have landed, as far as a half knows
        bool sat_out[2] = {false, false};
        for (int item = 0; item < 30; ++item) {
            const int tokens = from(0, 2) ? from(1, per_half) : from(1, 2 * per_half);
            const int past = from(0, 3) == 0 ? from(-40, 127) : from(0, short_items ? 900 : 3000);
            const int keys = std::max(0, past + tokens), all = keys <= kb ? 1 : (keys + kb - 1) / kb;
            const int block = from(0, 2) ? 0 : from(0, all - 1), blocks = from(0, 2) ? all - block : from(1, all - block);
            int count[2];
            half_blocks(past, tokens, per_half, kb, block, blocks, count);
            if (std::max(count[0], count[1]) != blocks) {
                std::printf("walk %d: blocks %d, halves %d and %d\n", walk, blocks, count[0], count[1]);
                return 1;
            }
            for (int h = 0; h < 2; ++h) {
                for (int j = 0; j < count[h]; ++j) {
                    if (j == 0 && scores_before_values(sat_out[h], count[h])) known[h] = std::max(known[h], base - 1);
                    if (base + j - ring > known[h]) {
                        std::printf("walk %d, item %d, half %d: waits for block %lld in %d slots and knows of block %lld\n", walk, item, h, base + j, ring, known[h]);
                        return 1;
                    }
                    behind += j == 0 && sat_out[h];
                    known[h] = std::max(known[h], base + j - 1);                 // by the block's scores
                }
                if (count[h] > 0) known[h] = std::max(known[h], base + count[h] - 1);      // by the last product
                sat_out[h] = count[h] < blocks;
            }
            base += blocks;
        }
    }
    std::printf("ok %ld\n", behind);
    return 0;
}
