// CPU model of scratch buffers leased on a handle that stands for a stream of
// each thread (torchvulkan_amd/csrc/scratch_pool.h, ThreadStream): what a thread
// queued on its own stream may still be pending when another thread leases.
// Prints "ok" and exits 0 on success; a violation ends it with a message.
#include "scratch_pool.h"

#include <cstdio>
#include <cstdlib>
#include <set>
#include <thread>

namespace {

#define CHECK(c, msg) do { if (!(c)) { std::fprintf(stderr, "scratch thread model: %s\n", msg); std::exit(1); } } while (0)

struct Model {
    typedef tvk::ThreadStream<int> Stream;
    int drains = 0;
    std::set<void*> live;
    void* alloc(size_t) { return *live.insert(std::malloc(1)).first; }
    void free(void* p) { live.erase(p); std::free(p); }
    void sync_device() { ++drains; }
    struct Capture { uint64_t id; };
    void* alloc_captured(size_t n) { return alloc(n); }
    bool keep(const Capture&, std::atomic<bool>*) { return true; }
};

typedef tvk::ScratchPool<Model> Pool;
typedef Model::Stream Stream;

// A call's lease: over as soon as its kernels are queued.
void* lease(Pool& pool, Stream s) {
    Pool::Buffer* b = pool.acquire(100, s);
    void* p = b->ptr;
    pool.release(b);
    return p;
}

void* of_thread(Pool& pool, int handle, bool each) {
    void* p = nullptr;
    std::thread([&] { p = lease(pool, Stream(handle, each)); }).join();
    return p;
}

}  // namespace

int main() {
    Model m;
    Pool pool(m, 1);
    // one handle, several threads: buffers of their own, the same one every time
    void* mine = lease(pool, Stream(2, true));
    CHECK(lease(pool, Stream(2, true)) == mine, "a thread's own stream order gives it its buffer again");
    void* other = of_thread(pool, 2, true);
    CHECK(other != mine, "two threads' streams share a buffer");
    void* third = of_thread(pool, 2, true);
    CHECK(third != mine && third != other, "a new thread takes over an ended one's stream");
    // an ordinary stream is one stream from any thread
    void* plain = lease(pool, Stream(7, false));
    CHECK(of_thread(pool, 7, false) == plain, "an ordinary stream has one buffer");
    CHECK(lease(pool, Stream(2, false)) != mine, "an ordinary handle is no thread's stream");
    // the same captured call
    Pool::Buffer* c = pool.acquire_captured(100, Stream(2, true), Model::Capture{5});
    pool.release(c);
    std::thread([&] {
        Pool::Buffer* d = pool.acquire_captured(100, Stream(2, true), Model::Capture{5});
        CHECK(d != c, "two threads' captured calls share a buffer");
        pool.release(d);
    }).join();
    // buffers of threads that have ended are given back after a drain, no others
    const size_t before = m.live.size();
    CHECK(m.drains == 0, "a lease drained the device");
    pool.trim_gone();
    CHECK(m.drains == 1 && m.live.size() == before - 2 && !m.live.count(other) && !m.live.count(third), "buffers of ended threads");
    CHECK(m.live.count(mine) && m.live.count(plain), "buffers of streams that are there");
    pool.trim_gone();
    CHECK(m.drains == 1, "nothing to give back, and a drain");
    std::puts("ok");
    return 0;
}
