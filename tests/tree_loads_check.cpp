// Every load of attention for trees, of every instance, head size, page size and place of a group: what it reads lies in its resource, and what it must not read is
// past it by either reading of a resource's bound: the lane's offset against what `more` leaves of the bytes, or the sum of both against the bytes.
#include <cstdint>
#include <cstdio>
#include <cstdlib>

#include "tree_loads.h"

using namespace egpt;

static const int kNowhere = static_cast<int>(0x80000000u);
static long checked = 0;

static void check(int offset, GroupLoad load, bool wanted, uint64_t at, const char* what) {
    const uint32_t by_lane = static_cast<uint32_t>(offset), left = load.bytes - static_cast<uint32_t>(load.more);
    const uint64_t sum = static_cast<uint64_t>(by_lane) + static_cast<uint32_t>(load.more);
    const bool dropped_by_lane = by_lane >= left, dropped_by_sum = sum >= load.bytes;
    const bool right = wanted ? !dropped_by_lane && !dropped_by_sum && sum == at && sum + 16 <= load.bytes
                              : dropped_by_lane && dropped_by_sum && load.more >= 0 && static_cast<uint32_t>(load.more) <= load.bytes;
    ++checked;
    if (!right) {
        std::printf("%s: lane offset %u, more %d, bytes %u, wanted %d at %llu\n", what, by_lane, load.more, load.bytes, wanted, static_cast<unsigned long long>(at));
        std::exit(1);
    }
}

int main() {
    const int pages[] = {16, 32, 48, 256, 4096, 1 << 20};
    for (int size = 2; size <= 4; size += 2)
        for (int instance = 64; instance <= 256; instance *= 2)
            for (int hd = 16 / size; hd <= instance; hd += 16 / size)
                for (int page : pages) {
                    if (static_cast<int64_t>(hd) * page * size > 0x7fffffff) continue;
                    const int row = instance * size, pieces = row / 16, keys = 1024 / row, loads = row / 64, key_bytes = hd * size;
                    for (int place = 0; place < 3; ++place) {
                        const int off = place == 0 ? 0 : place == 1 ? page - 16 : page / 32 * 16;
                        const uint32_t bytes = static_cast<uint32_t>(hd) * page * size - off * size;
                        for (int missing = 0; missing < 2; ++missing)
                            for (int load = 0; load < loads; ++load)
                                for (int lane = 0; lane < 64; ++lane) {
                                    const GroupLoad k = key_load(load, keys, key_bytes, missing);
                                    for (int piece = 0; piece < pieces; ++piece)
                                        check(key_lane(lane / pieces, key_bytes, piece, kNowhere), k, !missing && piece * 16 < key_bytes,
                                              static_cast<uint64_t>(load * keys + lane / pieces) * key_bytes + piece * 16, "keys");
                                    const int feature = load * (64 / size) + lane / size;
                                    const int piece = size == 2 ? lane % 2 ^ (feature >> 3 & 1) : lane % 4 ^ (feature >> 2 & 3);
                                    check(value_lane(lane, size, page, hd, kNowhere), value_load(load, size, page, hd, bytes, missing), !missing && feature < hd,
                                          static_cast<uint64_t>(feature) * page * size + piece * 16, "values");
                                }
                    }
                }
    std::printf("%ld places\n", checked);
    return 0;
}
