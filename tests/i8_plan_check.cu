// CPU check of how the 8-bit products' work is dealt out (built and run by tests/test_norm_i8.py): the kernel's own I8Plan, chunk sizes
// and item order (gg_i8.cuh, host-callable), for every pair of random launches.
//   * every (item, step) is covered by exactly one piece, no piece is empty, and pieces of an item agree on its first pair and their number;
//   * a cut item's pieces are its first pair's and the pairs' after it, one each, with workspace slots and counters of their own;
//   * chunks are not empty or larger than the limit, and the items of experts with and without rows, as a role's cursor finds them one after
//     the other, cover every (row, tile) once.
// Prints "ok <launches> <pieces>" and exits 0, or prints the first violation and exits 1.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <vector>

#include "gg_i8.cuh"

using namespace gg::moe;

#define CHECK(cond)                                                    \
    do {                                                               \
        if (!(cond)) {                                                 \
            std::printf("line %d: %s (items %d steps %d pairs %d)\n", __LINE__, #cond, items, steps, pairs); \
            std::exit(1);                                              \
        }                                                              \
    } while (0)

int main(int argc, char **argv) {
    const int launches = argc > 1 ? std::atoi(argv[1]) : 1000;
    uint64_t s = 88172645463325252ull;
    auto range = [&](int lo, int hi) {
        s ^= s << 13;
        s ^= s >> 7;
        s ^= s << 17;
        return lo + int(s % uint64_t(hi - lo + 1));
    };
    long long pieces_seen = 0, cut_seen = 0;
    for (int l = 0; l < launches; ++l) {
        const int pairs = range(0, 3) ? 74 : range(1, 80), steps = range(1, range(0, 1) ? 8 : 120);
        const int items = range(0, range(0, 1) ? 200 : 1000);
        const int most = 32 << range(0, 3);
        std::vector<std::vector<char>> done(items, std::vector<char>(steps, 0));
        std::map<int, std::vector<int>> owners;  // of cut items: the pairs, as they come
        std::map<int, std::pair<int, int>> told;
        std::set<int> slots;
        for (int c = 0; c < pairs; ++c) {
            const I8Plan plan(items, steps, most, pairs, c);
            cut_seen += plan.cut > 0 && plan.ranges > plan.cut;
            CHECK(plan.cut >= 0 && plan.cut <= items && plan.cut < 2 * pairs && plan.ranges <= pairs && (plan.ranges >= plan.cut || plan.ranges == pairs));
            plan.pieces([&](int item, int k0, int n, int first, int pieces) {
                ++pieces_seen;
                CHECK(item >= 0 && item < items && n > 0 && k0 >= 0 && k0 + n <= steps && pieces >= 1);
                for (int k = k0; k < k0 + n; ++k) {
                    CHECK(!done[item][k]);
                    done[item][k] = 1;
                }
                if (told.count(item))
                    CHECK(told[item].first == first && told[item].second == pieces);
                told[item] = {first, pieces};
                CHECK((pieces == 1) == (n == steps));
                if (pieces > 1) {
                    CHECK(c >= first && c < first + pieces && first + pieces <= pairs);
                    owners[item].push_back(c);
                    CHECK(slots.insert(2 * c + (c == first ? 1 : 0)).second);
                }
            });
        }
        std::set<int> counters;
        for (auto &o : owners) {
            CHECK(int(o.second.size()) == told[o.first].second);
            for (size_t i = 0; i < o.second.size(); ++i)
                CHECK(o.second[i] == told[o.first].first + int(i));
            CHECK(counters.insert(told[o.first].first).second);
        }
        for (auto &d : done)
            for (char c : d)
                CHECK(c);
        // chunks and item order of experts, some without rows, as a role with a stride sees them
        const int tiles = range(1, 40), experts = range(1, range(0, 1) ? 4 : 200), stride = range(1, 80);
        std::vector<int> start(experts + 1), first(experts + 1);
        for (int e = 0; e < experts; ++e) {
            const int count = range(0, 2) ? range(0, range(0, 1) ? 40 : 1500) : 0, chunks = i8_chunks(count, most);
            start[e + 1] = start[e] + count;
            first[e + 1] = first[e] + chunks;
            if (chunks) {
                const int size = i8_chunk_size(count, chunks);
                CHECK(size <= most && size % 32 == 0 && (chunks - 1) * size < count && chunks * size >= count);
            }
        }
        std::vector<char> rows_seen(size_t(start[experts]) * tiles, 0);
        for (int c = 0; c < stride; ++c) {
            I8Cursor cursor;
            for (int item = c; item < first[experts] * tiles; item += stride) {
                const I8Item it = cursor.at(item, tiles, experts, start.data(), first.data());
                CHECK(it.e >= 0 && it.e < experts && it.count > 0 && it.width >= it.count && it.width % 32 == 0 && it.width <= most);
                CHECK(it.r0 >= start[it.e] && it.r0 + it.count <= start[it.e + 1]);
                CHECK(it.n0 % kI8TileRows == 0 && it.n0 >= 0 && it.n0 / kI8TileRows < tiles);
                for (int r = it.r0; r < it.r0 + it.count; ++r) {
                    char &seen = rows_seen[size_t(r) * tiles + it.n0 / kI8TileRows];
                    CHECK(!seen);
                    seen = 1;
                }
            }
        }
        for (char c : rows_seen)
            CHECK(c);
    }
    if (cut_seen < launches)  // launches whose items are really cut are among them
        return std::printf("too few cut launches\n"), 1;
    std::printf("ok %d %lld\n", launches, pieces_seen);
    return 0;
}
