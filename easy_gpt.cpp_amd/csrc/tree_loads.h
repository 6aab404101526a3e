// Where the loads of attention for trees lie: plain arithmetic, which a program on the host can check as well.
//
// A load takes 16 bytes a lane by a resource that begins at a group of 16 keys (or their values) of one page and head and ends with it: at byte `offset` of a
// lane + `more`, the same for all lanes.  What must not be read ends up past the resource by the lane's offset alone: `more` never exceeds the resource's bytes, a lane
// past everything has the offset `nowhere`, and a load of nothing (a page that is missing, features past the head's) has no bytes and no `more`.
#pragma once

namespace egpt {

struct GroupLoad {
    int more;
    unsigned bytes;
};

// Load `load` of a group's keys has keys from load * keys on, key_bytes each; piece: the 16 bytes of the key that the lane takes.
constexpr int key_lane(int key, int key_bytes, int piece, int nowhere) { return piece * 16 < key_bytes ? key * key_bytes + piece * 16 : nowhere; }
constexpr GroupLoad key_load(int load, int keys, int key_bytes, bool missing) {
    return missing ? GroupLoad{0, 0u} : GroupLoad{load * keys * key_bytes, 16u * static_cast<unsigned>(key_bytes)};
}

// Load `load` of a group's values has features from load * (64 / size) on, of the group's 16 values 16 bytes a lane, which exchange places by the feature's number
// so that lanes that read them together read different banks; `bytes` from the group's first value to the head's end.
constexpr int value_lane(int lane, int size, int page_size, int hd, int nowhere) {
    const int feature = lane / size;
    const int piece = size == 2 ? lane % 2 ^ (feature >> 3 & 1) : lane % 4 ^ (feature >> 2 & 3);
    return feature < hd ? feature * page_size * size + piece * 16 : nowhere;
}
constexpr GroupLoad value_load(int load, int size, int page_size, int hd, unsigned bytes, bool missing) {
    const int feature = load * (64 / size);
    return missing || feature >= hd ? GroupLoad{0, 0u} : GroupLoad{feature * page_size * size, bytes};
}

}  // namespace egpt
