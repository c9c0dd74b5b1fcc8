// The pool's blocks under stream captures, with memory and captures made up: what tests/test_captured_memory.py builds and runs.
#include <cstdio>
#include <cstdlib>
#include <map>

#include "../sage_b200/csrc/runtime/runtime.h"

using namespace sage;

struct Made : DeviceMem {
    uint64_t now = 0;
    uintptr_t next = 1 << 20;
    int released = 0;
    std::map<uint64_t, std::shared_ptr<GoneGraphs>> told;
    void *alloc(size_t bytes) override {
        void *p = (void *)next;
        next += bytes;
        return p;
    }
    void release(void *) override { ++released; }
    uint64_t capture() override { return now; }
    void tell(uint64_t c, std::shared_ptr<GoneGraphs> g) override { told[c] = g; }
    void end(uint64_t c) {
        std::lock_guard<std::mutex> lock(told[c]->m);
        told[c]->captures.push_back(c);
        told[c]->any = true;
    }
};
#define CHECK(x)                                             \
    if (!(x)) {                                              \
        printf("line %d: %s is not so\n", __LINE__, #x);     \
        exit(1);                                             \
    }

static void follow(bool cache) {
    Made *m = new Made();
    {
        Allocator a(std::unique_ptr<DeviceMem>(m), 1ull << 40, cache);
        const auto during = [&](uint64_t c) {
            m->now = c;
            a.look();
        };
        const size_t n = 3 << 20;
        Block *warm = a.alloc(n);  // a call before the capture leaves its scratch in the pool
        char *scratch = warm->ptr;
        a.free(warm);
        during(7);
        Block *b = a.alloc(n);
        if (cache) CHECK(b->ptr == scratch);
        scratch = b->ptr;
        a.free(b);
        Block *again = a.alloc(n);  // the capture's next call works in the same memory
        CHECK(again->ptr == scratch);
        Block *result = a.alloc(700);  // a tensor made inside the capture and dropped behind it
        a.free(again);
        during(0);
        a.free(result);
        char *const result_at = result->ptr;
        Block *mine[64];
        for (Block *&t : mine) {  // calls and tensors from then on have other memory
            t = a.alloc(&t == mine ? n : 700);
            CHECK(t->ptr + t->size <= scratch || t->ptr >= scratch + n);
            CHECK(t->ptr != result_at);
        }
        during(9);  // as has another capture
        Block *other = a.alloc(n);
        CHECK(other->ptr + n <= scratch || other->ptr >= scratch + n);
        char *const second = other->ptr;
        a.free(other);
        a.free(mine[0]);  // an operand that is dropped while it is captured
        during(0);
        const uint64_t used = a.mem_used();
        a.release_cached();
        CHECK(a.mem_used() == used);
        m->end(7);
        a.look();
        CHECK(a.mem_used() < used);
        Block *back = a.alloc(n);  // the pool has the first graph's memory again, the second keeps its own
        if (cache) CHECK(back->ptr == scratch);
        Block *more = a.alloc(n);
        CHECK(more->ptr + n <= second || more->ptr >= second + n);
        during(11);  // a block of this capture that the next one is given back belongs to both
        Block *both = a.alloc(900);
        char *const shared = both->ptr;
        during(12);
        a.free(both);
        Block *fresh = a.alloc(900);
        CHECK(fresh->ptr != shared);
        during(0);
        m->end(12);
        a.look();
        Block *late = a.alloc(900);
        CHECK(late->ptr != shared);
        m->end(11);
        a.look();
        Block *freed = a.alloc(900);
        if (cache) CHECK(freed->ptr == shared);
        for (Block *t : {back, more, fresh, late, freed}) a.free(t);
        for (int i = 1; i < 64; ++i) a.free(mine[i]);
        m->end(9);
        a.look();
        CHECK(a.mem_used() == 0);
        during(20);  // a graph that still lives when the pool ends
        a.free(a.alloc(n));
        during(0);
    }
}

int main() {
    follow(true);
    follow(false);
    puts("fine");
    return 0;
}
