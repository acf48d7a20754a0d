// The ranges of the streaming attention's line (Shares in lq8_prefix_plan.cuh), on the CPU: reads cases
// "workers prefix_steps own_steps hand_out" from stdin and prints for each whether the ranges cover the line
// in order without an empty one, within 5 workers, whether owner() finds the range of every step, and
// the largest range: "ok ranges largest" or "bad <what> <range or step>".
#include "lq8_prefix_plan.cuh"

#include <cstdio>

using namespace lq;

int main() {
    int n, sp, so, chunks;
    while (scanf("%d %d %d %d", &n, &sp, &so, &chunks) == 4) {
        PrefixPlan p{};
        p.workers = n;
        p.workers_mul = ((1ull << 40) + n - 1) / n;
        p.sp = sp;
        p.chunks = chunks;
        const Shares s(p, so);
        const char* bad = nullptr;
        int where = 0, largest = 0;
        if (s.ranges > (chunks ? 5 : 1) * n) bad = "count";
        long long prefix = 0, own = 0;
        for (int c = 0; c < s.ranges && !bad; c++) {
            const int lo = s.start(c), hi = s.start(c + 1);
            if (c == 0 && lo != 0) bad = "first", where = c;
            if (hi <= lo) bad = "empty", where = c;
            largest = std::max(largest, hi - lo);
            for (int part = 0; part < 2; part++) {
                int a, b;
                s.range(c, part, a, b);
                if (a < b && part == 0 && a != prefix) bad = "prefix", where = c;
                if (a < b && part == 1 && a != own) bad = "own", where = c;
                if (a < b) (part ? own : prefix) = b;
            }
            for (int x : {lo, (lo + hi) / 2, hi - 1})
                if (!bad && s.owner(x) != c) bad = "owner", where = x;
        }
        if (!bad && (prefix != sp || own != so || (s.ranges > 0 && s.start(s.ranges) != sp + so))) bad = "end";
        if (bad) printf("bad %s %d\n", bad, where);
        else printf("ok %d %d\n", s.ranges, largest);
    }
    return 0;
}
