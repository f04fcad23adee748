// How many clusters of 2 .. 8 CTAs of a kernel a device holds at once: asked once per device, remembered once every answer is there. Host code without CUDA.
#pragma once
#include <mutex>

namespace b200q {
struct ClusterRoom {
    static constexpr int kMost = 8;
    // room[i]: clusters of i CTAs. ask(i, n) puts their number into n and returns 0 or an error, which comes back and leaves nothing behind: the next
    // call asks anew. (A number that is missing would be taken for no room, and the sums cut another way for the rest of the process.)
    template <typename Ask> int get(int device, Ask ask, const int** room) {
        std::lock_guard<std::mutex> lock(mu);
        int* c = count[device & 63];
        if (c[0] == 0) {
            for (int i = 2; i <= kMost; ++i)
                if (int rc = ask(i, c[i])) return rc;
            c[0] = 1;
        }
        *room = c;
        return 0;
    }

private:
    std::mutex mu;
    int count[64][kMost + 1] = {};
};
}  // namespace b200q
