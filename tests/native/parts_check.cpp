// The rows, slots and segments of psh_parts.h for offsets of any kind: nothing outside the arrays for those that make no
// sense, everything exactly once for those that ascend.  Offsets lie between two pages that cannot be read.
#include <sys/mman.h>
#include <unistd.h>

#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "psh_parts.h"

#define NEED(c)                                                                                                       \
    do {                                                                                                              \
        if (!(c)) {                                                                                                   \
            std::printf("%s:%d: %s  (trial %d: n %d rows %d L %d policies %d)\n", __FILE__, __LINE__, #c, trial, n, rows, L, P); \
            std::exit(1);                                                                                             \
        }                                                                                                             \
    } while (0)

template <class F> static int search(int n, int slot, F key) {   // what the 64 lanes of a wave do
    Search s{0, n + 1};
    while (s.count > 1) {
        uint64_t below = 0;
        for (int lane = 0; lane < 64; ++lane)
            if (s.probes(lane) && key(s.candidate(lane)) <= slot) below |= 1ull << lane;
        s.narrow(below);
    }
    return s.lo;
}

struct Fenced {   // an int array that ends where a page ends, in front of one that cannot be touched; `front`: begins behind one
    int* p;
    explicit Fenced(int n, bool front) {
        const size_t page = sysconf(_SC_PAGESIZE), bytes = ((size_t)n * 4 + page - 1) / page * page;
        char* const m = (char*)mmap(nullptr, bytes + 2 * page, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
        if (m == MAP_FAILED || mprotect(m + page, bytes, PROT_READ | PROT_WRITE)) std::abort();
        base = m;
        size = bytes + 2 * page;
        p = (int*)(front ? m + page : m + page + bytes - (size_t)n * 4);
    }
    ~Fenced() { munmap(base, size); }
    char* base;
    size_t size;
};

int main(int argc, char** argv) {
    const int trials = argc > 1 ? std::atoi(argv[1]) : 1000;
    std::mt19937 rng(7);
    const auto upto = [&](int lo, int hi) { return (int)(lo + (int64_t)(rng() % (uint64_t)((int64_t)hi - lo + 1))); };
    for (int trial = 0; trial < trials; ++trial) {
        const int n = trial % 3 == 0 ? upto(1, 5) : upto(1, 300), TS = trial % 2 ? 8 : 16;
        const bool huge = trial % 11 == 0;
        const int rows = huge ? (1 << 30) - upto(0, 5) : upto(0, trial % 5 ? 400 : 9000);
        const int L = huge ? TS << upto(18, 24) : TS * upto(1, trial % 4 ? 12 : 2000), P = upto(1, n + 2);
        const bool ascend = trial % 2 == 0;
        Fenced off(n + 1, trial % 7 < 3), grp(P + 1, trial % 7 < 3);
        const auto fill = [&](int* p, int count, int top) {
            std::vector<int> v(count);
            for (auto& o : v) o = upto(0, top);
            if (ascend) std::sort(v.begin(), v.end());
            for (int i = 0; i < count; ++i) p[i] = v[i];
            if (ascend) p[0] = 0;
            else
                for (int k = 0; k < 3; ++k) p[upto(0, count - 1)] = (int[]){-1, INT32_MIN, INT32_MAX, top + 1, -1000}[upto(0, 4)];
        };
        fill(off.p, n + 1, rows);
        fill(grp.p, P + 1, n);
        const Parts parts{off.p, n, rows, L};
        const int64_t slots = parts_slots(rows, n, L), checks = parts_slots(rows, n, TS);
        std::vector<char> seen(huge ? 0 : rows, 0);
        std::vector<int> pieces(n + 1, 0);
        NEED(slots < INT32_MAX);
        for (int slot = 0; slot < slots; ++slot) {
            const int part = search(n, slot, [&](int i) { NEED(i >= 0 && i <= n); return parts.first_slot(i); });
            NEED(part >= 0 && part <= n);
            const Piece q = piece_of(parts, part, parts.at(part), parts.at(part + 1), slot);
            NEED(q.j >= 0 && q.begin >= 0 && q.begin <= rows && q.end <= rows && q.part_begin >= 0 && q.part_end <= rows);
            if (q.begin >= q.end && q.j > 0) continue;
            ++pieces[part];
            if (part < n) {   // the stored states of its tiles
                const int64_t c = check_slot(q, TS), tiles = q.begin < q.end ? ((int64_t)q.end - q.begin + TS - 1) / TS : 0;
                NEED(c >= 0 && c + (tiles > 0 ? tiles - 1 : 0) < checks);
            }
            if (ascend && !huge)
                for (int r = q.begin; r < q.end; ++r) {
                    NEED(!seen[r] && r >= q.part_begin && r < q.part_end);
                    seen[r] = 1;
                }
        }
        for (const CutPlaces by : {CutPlaces{true}, CutPlaces{false}, cut_places(rows, n, L)}) {   // places of the pieces of parts that are cut
            const int64_t count = by.by_rows ? places_by_rows(rows, L) : slots;
            NEED(count >= cut_places_count(rows, n, L));
            std::vector<char> taken(count, 0);
            for (int i = 0; i < n; ++i) {
                const int b = parts.at(i), e = parts.at(i + 1);
                if (e - b <= L) continue;
                for (int j = 0; j < piece_count(b, e, L); ++j) {
                    const int64_t at = by.first(parts, i, b) + j;
                    NEED(at >= 0 && at < count && !(ascend && taken[at]));
                    taken[at] = 1;
                }
            }
        }
        for (int i = 0; i < n; ++i) {   // pieces that are joined
            const int b = parts.at(i), e = parts.at(i + 1);
            if (e - b > L) NEED(parts.first_slot(i) + (int64_t)piece_count(b, e, L) <= slots);
            if (ascend) NEED(pieces[i] == (e - b > L ? piece_count(b, e, L) : 1));
        }
        if (ascend)
            for (char s : seen) NEED(s);
        // policies of the sequences
        const Shares share{grp.p, P, n};
        for (int s = 0; s < n; ++s) {
            const int p = P == 1 ? 0 : search(P - 1, s, [&](int i) { NEED(i >= 0 && i < P); return share.at(i); });
            NEED(p >= 0 && p < P);
            if (ascend) NEED(share.at(p) <= s && s < share.at(p + 1));
        }
        // sums over the slots of a policy
        for (int seg : {0, 1, 32, 64}) {
            const PolicySlots a{parts, share, seg};
            const int64_t segs = seg ? policy_segments(slots, P, seg) : 0;
            std::vector<char> written(seg ? segs : 0, 0), added(slots, 0);
            for (int k = 0; k < segs; ++k) {
                const int p = P == 1 ? 0 : search(P - 1, k, [&](int i) { NEED(i >= 0 && i < P); return a.seg_of(i); });
                NEED(p >= 0 && p < P);
                int64_t begin, stop;
                if (!a.segment(k, p, begin, stop)) continue;
                NEED(begin >= 0 && stop <= slots);
                written[k] = 1;
                for (int64_t s = begin; s < stop; ++s) {
                    if (ascend) NEED(!added[s]);
                    added[s] = 1;
                }
            }
            for (int p = 0; p < P; ++p) {
                int first, count;
                a.of_policy(p, first, count);
                NEED(first >= 0 && count >= 0 && first + (int64_t)count <= (seg ? segs : slots));
                if (ascend && seg)
                    for (int k = first; k < first + count; ++k) NEED(written[k]);
            }
            if (ascend && seg)
                for (int64_t s = 0; s < slots; ++s) NEED(added[s] == (s < parts.first_slot(n)));
        }
    }
    std::puts("ok");
}
