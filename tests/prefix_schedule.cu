// Host model of how the bf16 shared-prefix attention hands out its work, on the library's own cut
// (plan_cut, Line, flow_range, OwnSteps) and rule (hand_out): per CTA the batches of up to 16 items
// that the scheduler puts into the flows' rings of two, and the warps that take a round of each
// flow in turn. Reads cases from stdin, a line each:
//   rule rows_per_seq heads kv_heads prefix max_q max_kv n_seqs kv[0] .. kv[n_seqs - 1]
// (rule 0: the library's; 1: a flow out of steps gets its missing rounds only at the end) and
// prints per case how many CTAs end up waiting for themselves, the first of them (-1), and "bad"
// where the flows' rounds or the items' tiles do not add up.
#include "lq8_prefix_plan.cuh"

#include <cstdio>
#include <utility>
#include <vector>

using namespace lq;

struct Put {
    int flow;
    int rounds;
};

struct Model {
    PrefixAttnArgs a{};
    PagedSeqs s{};
    PrefixPlan p{};
    std::vector<SeqInfo> seqs;
    std::vector<std::pair<int, int>> items;  // own items in order: (tiles, steps)
    int own_steps = 0;
    long long tiles = 0;

    void cut() {
        const OwnSteps os{a, p};
        for (const SeqInfo& i : seqs)
            for (int kh = 0; kh < a.n_kv; kh++)
                for (int rb = 0; rb < os.blocks(i); rb++) {
                    items.push_back({os.tiles(i, rb), os.steps(i, rb)});
                    own_steps += os.steps(i, rb);
                }
    }

    // what the scheduler of CTA c puts into the rings; the flows' rounds in all
    std::vector<Put> puts(int c, int rule, long long total[2]) {
        std::vector<Put> out;
        const Line line(p, own_steps, p.pair_p, p.pair_o);
        total[0] = total[1] = 0;
        for (int own = 0; own < 2; own++) {
            if (!own && line.sp == 0) continue;
            const bool paired = own ? p.pair_o : p.pair_p;
            const long long n_items = own ? (long long)items.size() : (long long)a.n_kv * p.n_rb;
            int step[2], hi[2], rounds[2] = {0, 0};
            long long j[2] = {0, 0};
            int t[2] = {0, 0};
            for (int f = 0; f < 2; f++) {
                flow_range(line, paired, c, f, own, step[f], hi[f]);
                if (step[f] >= hi[f]) continue;
                int rest = step[f];
                while (rest >= (own ? items[j[f]].second : p.np)) rest -= own ? items[j[f]++].second : (j[f]++, p.np);
                t[f] = rest;
            }
            for (bool first = true; step[0] < hi[0] || step[1] < hi[1]; first = false) {
                bool go[2];
                const bool live[2] = {step[0] < hi[0], step[1] < hi[1]};
                const int had[2] = {rounds[0], rounds[1]};
                for (int f = 0; f < 2; f++) {
                    HandOut h = hand_out(f, first, live[f], live[f ^ 1], had[f], had[f ^ 1]);
                    if (paired) h = HandOut{live[f], 0};
                    if (rule == 1) h.idle = 0;
                    go[f] = h.go;
                    if (h.idle > 0) {
                        out.push_back({f, h.idle});
                        rounds[f] += h.idle;
                    }
                }
                for (int f = 0; f < 2; f++) {
                    if (!go[f]) continue;
                    int n = 0;
                    for (int k = 0; k < 16 && step[f] < hi[f] && j[f] < n_items; k++, j[f]++, t[f] = 0) {
                        const int nt = own ? items[j[f]].first : p.np, ns = own ? items[j[f]].second : p.np;
                        const int take = std::min(ns - t[f], hi[f] - step[f]);
                        n += std::max(0, std::min(nt, t[f] + take) - std::min(t[f], nt));
                        step[f] += take;
                        if (step[f] >= hi[f]) break;
                    }
                    if (j[f] >= n_items) hi[f] = step[f];
                    if (n > 0) out.push_back({f, n});
                    rounds[f] += n;
                    tiles += paired && f ? 0 : n;
                }
            }
            if (!paired && rounds[0] != rounds[1]) {
                const int f = rounds[0] < rounds[1] ? 0 : 1, more = std::abs(rounds[0] - rounds[1]);
                out.push_back({f, more});
                rounds[f] += more;
            }
            total[0] += rounds[0];
            total[1] += rounds[1];
        }
        out.push_back({0, 0});  // the end
        out.push_back({1, 0});
        return out;
    }

    // whether the rounds get done: batch k of a flow is put when the serving warps have begun its
    // batch k - 1 (or wait for it); they take flow 0 and flow 1 in turn and wait where there is none
    static bool ends(const std::vector<Put>& puts) {
        std::vector<int> batch[2];
        int begun[2] = {0, 0}, left[2] = {0, 0};  // batches asked for; rounds left of the one begun
        bool waits = false, ended[2] = {false, false};
        int f = 0;
        auto serve = [&]() {
            while (!(ended[0] && ended[1])) {
                if (!ended[f]) {
                    if (left[f] == 0) {
                        if (!waits) begun[f]++;
                        waits = (int)batch[f].size() < begun[f];
                        if (waits) return;
                        left[f] = batch[f][begun[f] - 1];
                        ended[f] = left[f] == 0;
                    }
                    if (!ended[f]) left[f]--;
                }
                f ^= 1;
            }
        };
        serve();
        for (const Put& u : puts) {
            const int k = (int)batch[u.flow].size();
            if (k >= 2 && begun[u.flow] < k) return false;
            batch[u.flow].push_back(u.rounds);
            serve();
        }
        return ended[0] && ended[1];
    }
};

int main() {
    int rule, q, heads, kv_heads, prefix, max_q, max_kv, n;
    while (scanf("%d %d %d %d %d %d %d %d", &rule, &q, &heads, &kv_heads, &prefix, &max_q, &max_kv, &n) == 8) {
        Model m;
        m.a.n_heads = heads, m.a.n_kv = kv_heads, m.a.group = heads / kv_heads;
        m.a.group_mul = ((1ull << 36) + m.a.group - 1) / m.a.group;
        m.a.prefix_len = prefix, m.a.max_q = max_q, m.a.max_kv = max_kv;
        m.s.n_seqs = n, m.s.rows = n * q;
        for (int b = 0; b < n; b++) {
            int kv;
            if (scanf("%d", &kv) != 1) return 1;
            m.seqs.push_back(SeqInfo{b * q, q, kv});
        }
        if (plan_cut(m.a, m.s, false, 148, &m.p) >= PREFIX_MAX_STEPS) {
            printf("refused\n");
            continue;
        }
        m.cut();
        int stuck = 0, at = -1;
        bool bad = false;
        for (int c = 0; c < m.p.workers; c++) {
            long long total[2];
            const std::vector<Put> puts = m.puts(c, rule, total);
            bad = bad || total[0] != total[1];
            if (!Model::ends(puts)) {
                if (!stuck++) at = c;
            }
        }
        long long want = (long long)m.p.sp;
        for (const auto& i : m.items) want += i.first;
        bad = bad || want != m.tiles;
        printf("%d %d%s\n", stuck, at, bad ? " bad" : "");
    }
    return 0;
}
