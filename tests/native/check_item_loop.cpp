/* The prompt attention kernel's item loop (item_loop.h) with threads for a tile's four warps.
 * Every warp's wait for an item may run out, once and for good, whatever the others' do; the
 * work of an item is a barrier of all four.  No warp may be left at a barrier: a barrier that is
 * not complete after `limit` counts as a hang (the threads leave it, so this program ends).
 *
 * argv[1]: "loop" the kernel's loop, "alone" one whose warps leave by themselves (which has
 * to be seen to hang).  Prints "OK <mode> <hangs>"; exit code 1 where that is not as it should be. */
#include <atomic>
#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <thread>
#include <vector>

#include "../../glint_b200/csrc/item_loop.h"

namespace {

constexpr int kWarps = 4;

/* barrier with a reduction, as barrier.cta.red.or */
struct Barrier {
    std::mutex mu;
    std::condition_variable cv;
    int arrived = 0, phase = 0;
    bool acc = false, result = false;
    std::atomic<bool> hung{false};
    bool any(bool p, std::chrono::milliseconds limit)
    {
        std::unique_lock<std::mutex> lk(mu);
        if (hung)
            return true;
        acc |= p;
        if (++arrived == kWarps) {
            result = acc, acc = false, arrived = 0, ++phase;
            cv.notify_all();
            return result;
        }
        const int mine = phase;
        if (!cv.wait_for(lk, limit, [&] { return phase != mine || hung; })) {
            hung = true;
            cv.notify_all();
        }
        return hung ? true : result;
    }
};

/* warp w's wait runs out at item fail[w] (or never, -1); items end at `last` */
bool hangs(const int (&fail)[kWarps], int last, bool alone)
{
    Barrier bar;
    const auto limit = std::chrono::milliseconds(alone ? 200 : 5000);
    std::vector<std::thread> warps;
    for (int w = 0; w < kWarps; ++w)
        warps.emplace_back([&, w] {
            bool alive = true;
            auto next = [&](int i) {
                alive = alive && i != fail[w];
                return alive && i < last && !bar.hung;
            };
            auto any = [&](bool p) { return bar.any(p, limit); };
            auto work = [&](int) { any(false); };
            if (!alone) {
                glint::item_loop(next, any, work);
            } else {
                for (int i = 0; next(i); ++i)
                    work(i);
            }
        });
    for (auto &t : warps)
        t.join();
    return bar.hung;
}

} // namespace

int main(int argc, char **argv)
{
    const bool alone = argc > 1 && !strcmp(argv[1], "alone");
    int count = 0;
    const int last = 2;
    for (int n = 0; n < 256; ++n) { /* every warp at item 0, 1, 2 (the end's own wait) or never */
        int fail[kWarps];
        for (int w = 0; w < kWarps; ++w)
            fail[w] = (n >> (2 * w) & 3) == 3 ? -1 : (n >> (2 * w) & 3);
        if (alone && n % 37 != 0) /* a hang costs its limit: a few are enough */
            continue;
        count += hangs(fail, last, alone);
    }
    printf("%s %s %d\n", (count > 0) == alone ? "OK" : "WRONG", alone ? "alone" : "loop", count);
    return (count > 0) == alone ? 0 : 1;
}
