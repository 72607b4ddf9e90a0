// Cuts the work of random ragged calls into shares with the library's own schedule, block by block of the launch, and checks
// that every block of keys of every row tile is taken once, in order, that no piece is empty, and that the first piece of a
// cut tile names the shares that hold the others.  Prints "ok" and the number of cut tiles.
#include <algorithm>
#include <cstdio>
#include <map>
#include <random>
#include <vector>

#include "../eptq_b200/csrc/attention_schedule.cuh"

using namespace eptq;

static std::mt19937 generator(1);
static int from(int a, int b) { return a + static_cast<int>(generator() % static_cast<unsigned>(b - a + 1)); }

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s (call %d)\n", __LINE__, #x, call); return 1; } } while (0)

int main() {
    const int tiles_tokens[] = {256, 128, 64, 32, 16, 8, 4, 2, 36, 84, 6, 254, 50, 1};
    long cut_tiles = 0;
    for (int call = 0; call < 6000; ++call) {
        const int tile = tiles_tokens[from(0, 13)], groups = from(1, 9), batch = from(1, 6), shares = from(1, 148), kb = from(0, 1) ? 128 : 64;
        CutRule rule{from(1, 12), from(0, 3), from(1, 6), from(0, 3)};
        std::vector<Request> requests;
        std::vector<long long> cost;
        long long all = 0;
        for (int b = 0; b < batch; ++b) {
            const int n = from(0, 3) == 0 ? 0 : from(0, 1) ? from(1, 5) : from(1, 700);
            const int kv = from(0, 3) == 0 ? from(0, n) : n + (from(0, 1) ? from(0, 300) : from(0, 6000));
            const Request r = request_from(0, n, 1000, kv, 1 << 20, true);
            CHECK(r.n == n && r.past == kv - n);
            long long sum = 0;
            const int tiles = tiles_of(r, tile);
            CHECK(tiles == (n + tile - 1) / tile);
            for (int i = 0; i < tiles; ++i) {
                CHECK(blocks_before(r, tile, kb, i) == sum);
                const int keys = r.past + std::min(n, (i + 1) * tile);
                CHECK(blocks_of(r, tile, kb, i) == std::max(1, (keys + kb - 1) / kb));
                sum += blocks_of(r, tile, kb, i);
            }
            CHECK(blocks_before(r, tile, kb, tiles) == sum);
            requests.push_back(r);
            cost.push_back((sum + static_cast<long long>(tiles) * rule.tile) * groups);
            all += cost.back();
        }
        if (all == 0) continue;
        const long long size = share_of(all, shares, rule);
        auto place = [&](long long x) {
            int b = 0;
            while (x >= cost[b]) x -= cost[b++];
            return place_of(requests[b], tile, kb, rule, x, [&](int lo, int hi, long long y) {
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (cost_before(requests[b], tile, kb, rule, mid) <= y) lo = mid; else hi = mid - 1;
                }
                return lo;
            });
        };
        auto cut = [&](int c) -> long long {
            const long long x = c * size;
            if (c == shares || x >= all) return all;
            Place p = place(x);
            return moved(p, rule, x);
        };
        std::map<long long, std::vector<int>> pieces;
        std::map<long long, std::pair<int, int>> named;
        long long at = 0;
        for (int c = 0; c < shares; ++c) {
            const long long begin = cut(c), end = cut(c + 1);
            CHECK(begin == at && end >= begin);
            at = end;
            for (long long x = begin; x < end;) {
                const Place p = place(x);
                CHECK(p.ahead == 0 || p.ahead == rule.tile);
                x += p.ahead;
                const long long take = std::min<long long>(end - x, p.blocks - p.block);
                CHECK(take > 0);
                const long long tile_begin = x - p.block, tile_end = tile_begin + p.blocks;
                if (take < p.blocks) {
                    pieces[tile_begin].push_back(c);
                    if (p.block == 0) named[tile_begin] = {c, last_share(tile_end, size, rule)};
                }
                x += take;
            }
        }
        CHECK(at == all);
        for (const auto& piece : pieces) {
            const auto n = named.find(piece.first);
            CHECK(n != named.end());
            const std::vector<int>& held = piece.second;
            CHECK(held.front() == n->second.first && held.back() == n->second.second && static_cast<int>(held.size()) == n->second.second - n->second.first + 1);
            ++cut_tiles;
        }
    }
    std::printf("ok %ld\n", cut_tiles);
    return 0;
}
