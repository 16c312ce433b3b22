// pages_check.cpp -- gbx::PageTable against a model of it that keeps every
// token: random appends, forks, truncations, releases and compactions, with the
// copies carried out on an array of page contents.  Prints "ok" and the number
// of steps, or the first thing that is wrong.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <vector>

#include "gbx_model.hpp"

#define CHECK(x)                                                       \
    do {                                                               \
        if (!(x)) {                                                    \
            std::printf("wrong at step %d: %s\n", step, #x);           \
            return 1;                                                  \
        }                                                              \
    } while (0)

int main(int argc, char** argv)
{
    const int pages = std::atoi(argv[1]), P = std::atoi(argv[2]), steps = std::atoi(argv[3]);
    std::mt19937 rng((unsigned)std::atoi(argv[4]));
    gbx::PageTable t(pages, P);
    std::vector<std::vector<int>> content(pages, std::vector<int>(P, -1));   // the "device"
    std::map<int, std::vector<int>> want;                                    // tokens of each sequence
    int next = 0;
    auto copy = [&](const gbx::PageTable::Copies& c) {
        // as the kernel may: every source read before any target is written, no target a source, none twice
        std::set<int> src(c.src.begin(), c.src.end()), dst(c.dst.begin(), c.dst.end());
        if (dst.size() != c.dst.size()) return false;
        for (int d : dst)
            if (src.count(d)) return false;
        for (size_t i = 0; i < c.src.size(); ++i) content[c.dst[i]] = content[c.src[i]];
        return true;
    };
    for (int step = 0; step < steps; ++step) {
        const int op = (int)(rng() % 10);
        std::vector<int> ids;
        for (auto& kv : want) ids.push_back(kv.first);
        if (op == 0 || ids.empty()) {
            const int id = t.newSequence();
            CHECK(!want.count(id));
            want[id] = {};
        } else if (op == 1) {
            const int from = ids[rng() % ids.size()], id = t.fork(from);
            CHECK(id >= 0 && !want.count(id));
            want[id] = want[from];
        } else if (op == 2) {
            const int id = ids[rng() % ids.size()];
            CHECK(t.release(id));
            CHECK(!t.release(id) && t.fork(id) == -1 && t.length(id) == -1);
            want.erase(id);
        } else if (op == 3) {
            const int id = ids[rng() % ids.size()];
            const int64_t keep = (int64_t)(rng() % (want[id].size() + 1));
            CHECK(!t.truncate(id, (int64_t)want[id].size() + 1) && !t.truncate(id, -1));
            CHECK(t.truncate(id, keep));
            want[id].resize((size_t)keep);
        } else if (op == 4) {
            const gbx::PageTable::Copies c = t.compact();
            CHECK(copy(c));
            for (int64_t p = 0; p < t.pages(); ++p) CHECK((t.references(p) > 0) == (p < t.pages() - t.freePages()));
        } else {
            std::shuffle(ids.begin(), ids.end(), rng);
            ids.resize(1 + rng() % ids.size());
            std::vector<int> n;
            for (size_t i = 0; i < ids.size(); ++i) n.push_back((int)(rng() % (2 * P + 2)));
            gbx::PageTable::Copies c, none;
            std::vector<int> twice = ids, n2 = n;
            twice.push_back(ids[0]);
            n2.push_back(1);
            const int64_t free0 = t.freePages();
            CHECK(!t.append(twice, n2, &none) && none.src.empty() && t.freePages() == free0);
            CHECK(!t.append({12345}, {1}, &none));
            if (!t.append(ids, n, &c)) {
                CHECK(c.src.empty() && t.freePages() == free0);
                for (int id : ids) CHECK(t.length(id) == (int64_t)want[id].size());
            } else {
                CHECK(copy(c));
                for (size_t i = 0; i < ids.size(); ++i)
                    for (int k = 0; k < n[i]; ++k) {
                        const int64_t at = (int64_t)want[ids[i]].size();
                        const int page = t.pagesOf(ids[i])[at / P];
                        CHECK(t.references(page) == 1);   // nobody else's page is written to
                        content[page][at % P] = next;
                        want[ids[i]].push_back(next++);
                    }
            }
        }
        // every token is where the table says, every page is counted
        std::vector<int> refs(pages, 0);
        for (auto& kv : want) {
            CHECK(t.length(kv.first) == (int64_t)kv.second.size());
            const std::vector<int32_t>& list = t.pagesOf(kv.first);
            CHECK((int64_t)list.size() == ((int64_t)kv.second.size() + P - 1) / P);
            for (int32_t p : list) ++refs[p];
            for (size_t k = 0; k < kv.second.size(); ++k) CHECK(content[list[k / P]][k % P] == kv.second[k]);
        }
        int64_t used = 0;
        for (int p = 0; p < pages; ++p) {
            CHECK(refs[p] == t.references(p));
            used += refs[p] > 0;
        }
        CHECK(t.freePages() == pages - used);
    }
    std::printf("ok %d\n", steps);
    return 0;
}
