// session_check.cpp -- gbx::Session and gbx::PageTable from C++, where the C ABI
// does not reach: page sizes that cannot be (mode "sizes", no GPU), and loading a
// model again under an open session (mode "reload", a GGUF's path).
// Prints "ok", or what is wrong.
#include <cstdio>
#include <cstring>

#include "gbx_model.hpp"

#define CHECK(x)                           \
    do {                                   \
        if (!(x)) {                        \
            std::printf("wrong: %s\n", #x); \
            return 1;                      \
        }                                  \
    } while (0)

static int sizes()
{
    for (int size : {0, -16}) {
        gbx::PageTable t(4, size);
        const int s = t.newSequence();
        gbx::PageTable::Copies c;
        CHECK(t.freePages() == 0 && t.pages() == 0);
        CHECK(t.truncate(s, 0) && !t.truncate(s, 1));
        CHECK(!t.append({s}, {1}, &c) && t.append({s}, {0}, &c));
        CHECK(t.compact().src.empty() && t.release(s));
        gbx::TransformerModel model;   // not loaded: the session does not open
        gbx::Session session(model, 4, size);
        const int x = session.newSequence();
        CHECK(!session.ok() && session.truncate(x, 0) && session.forward({x}, {1}, {1}).empty());
    }
    return 0;
}

static int reload(const char* path)
{
    gbx::TransformerModel model;
    CHECK(model.loadModel(path));
    gbx::Session s(model, 8, 16);
    CHECK(s.ok());
    const int x = s.newSequence();
    CHECK(s.nextTokens({x}, {1, 2, 3}, {3}, 0.0, {}).size() == 1);
    // a model is loaded once: refused, and the session goes on over the weights it was opened on
    CHECK(!model.loadModel(path));
    gbx::Session t(model, 8, 16);
    const int y = t.newSequence();
    CHECK(t.ok() && t.nextTokens({y}, {1, 2, 3}, {3}, 0.0, {}).size() == 1);
    const std::vector<float> a = s.forward({x}, {4}, {1}), b = t.forward({y}, {4}, {1});
    CHECK(!a.empty() && a.size() == b.size() && !std::memcmp(a.data(), b.data(), a.size() * sizeof(float)));
    CHECK(s.compact() == 0 && s.length(x) == 4);
    return 0;
}

int main(int argc, char** argv)
{
    const int rc = argc > 2 && !std::strcmp(argv[1], "reload") ? reload(argv[2]) : sizes();
    if (!rc) std::printf("ok\n");
    return rc;
}
