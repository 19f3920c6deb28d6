// Growth of scratch that a call can do without (grow_scratch), against a device with a given amount of room.
#include <cstdio>
#include <random>
#include <vector>

#include "host_logic.hpp"

#define CHECK(x)                                                     \
    do {                                                             \
        if (!(x)) {                                                  \
            std::printf("line %d: %s\n", __LINE__, #x);              \
            return 1;                                                \
        }                                                            \
    } while (0)

struct Device {
    explicit Device(uint64_t r) : room(r) {}
    uint64_t room, have = 0, refused = UINT64_MAX;
    std::vector<uint64_t> asked;
    bool grow(uint64_t wanted, uint64_t limit) {
        asked.clear();
        return psi::grow_scratch(wanted, have, limit, refused, [&](uint64_t bytes) {
            asked.push_back(bytes);
            if (have + bytes > room) return false;  // both exist for a moment
            have = bytes;
            return true;
        });
    }
};

int main() {
    Device d{10000};
    CHECK(d.grow(1000, 8000) && d.have == 1500 && d.asked.size() == 1);
    CHECK(d.grow(1500, 8000) && d.asked.empty());
    CHECK(d.grow(6000, 8000) && d.have == 8000 && d.asked == std::vector<uint64_t>({8000}));  // half more, cut at the limit
    CHECK(!d.grow(8001, 8000) && d.asked.empty() && d.have == 8000);
    CHECK(d.grow(8000, 8000) && d.asked.empty());
    Device e{10000};
    CHECK(e.grow(2000, 1 << 20) && e.have == 3000);
    CHECK(e.grow(6000, 1 << 20) && e.have == 6000 && e.asked == std::vector<uint64_t>({9000, 6000}));  // no room for half more
    CHECK(!e.grow(7000, 1 << 20) && e.asked.size() == 2 && e.have == 6000);                         // the old one stays
    CHECK(!e.grow(7000, 1 << 20) && e.asked.empty());                                               // and nothing is asked for again
    CHECK(!e.grow(9000, 1 << 20) && e.asked.empty());
    CHECK(e.grow(6000, 1 << 20) && e.grow(10, 1 << 20) && e.asked.empty());
    CHECK(!e.grow(6500, 1 << 20) && e.asked == std::vector<uint64_t>({6500}) && e.refused == 6500);  // half more is known not to be there
    // random: never above the limit, never without what is asked for, never more than two questions, none for a size that was refused
    std::mt19937_64 rng(1);
    for (int round = 0; round < 2000; ++round) {
        Device x{rng() % 100000};
        const uint64_t limit = 1 + rng() % 60000;
        for (int step = 0; step < 30; ++step) {
            const uint64_t wanted = 1 + rng() % 70000, before = x.have, refused = x.refused;
            const bool got = x.grow(wanted, limit);
            CHECK(x.have <= limit && x.have >= before && got == (x.have >= wanted && wanted <= limit));
            CHECK(x.asked.size() <= 2);
            for (uint64_t a : x.asked) CHECK(a < refused && a >= wanted);
        }
    }
    std::puts("scratch ok");
    return 0;
}
