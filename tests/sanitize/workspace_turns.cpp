// workspace_turns.cpp — the per-stream workspaces (tq_capi.cpp) among host
// threads, on a stand-in for the HIP runtime: device memory is host memory, so
// AddressSanitizer sees a buffer that is used after it was freed
// (tests/test_workspace_turns.py).
//
//   workspace_turns release    a release while another thread has a buffer
//   workspace_turns evict      more streams than are cached, likewise
//   workspace_turns threads    hipStreamPerThread: a stream of each thread's
#include <hip/hip_runtime.h>

#include <atomic>
#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <set>
#include <thread>
#include <vector>

#include "tq_internal.h"

// ---- the stand-in ----------------------------------------------------------
namespace {
std::atomic<bool> g_idle{true};  // every stream's work is done
std::mutex g_mu;
std::set<void*> g_live;  // allocations
struct Event {
    std::thread::id by;  // the thread that recorded it
    hipStream_t on;
};
thread_local hipError_t t_error = hipSuccess;
hipError_t done(hipError_t e) {
    if (e != hipSuccess) t_error = e;
    return e;
}
}  // namespace

extern "C" {
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetLastError(void) {
    const hipError_t e = t_error;
    t_error = hipSuccess;
    return e;
}
hipError_t hipMalloc(void** p, size_t n) {
    *p = std::malloc(n);
    std::lock_guard<std::mutex> lock(g_mu);
    g_live.insert(*p);
    return hipSuccess;
}
hipError_t hipFree(void* p) {
    {
        std::lock_guard<std::mutex> lock(g_mu);
        g_live.erase(p);
    }
    std::free(p);
    return hipSuccess;
}
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
    *s = hipStreamCaptureStatusNone;
    return hipSuccess;
}
// hipStreamPerThread is the calling thread's stream: idle unless it is the worker's.
thread_local bool t_has_work = false;
hipError_t hipStreamQuery(hipStream_t s) {
    return done(g_idle || (s == hipStreamPerThread && !t_has_work) ? hipSuccess : hipErrorNotReady);
}
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) {
    *e = reinterpret_cast<hipEvent_t>(new Event{});
    return hipSuccess;
}
hipError_t hipEventRecord(hipEvent_t e, hipStream_t s) {
    *reinterpret_cast<Event*>(e) = Event{std::this_thread::get_id(), s};
    return hipSuccess;
}
hipError_t hipEventQuery(hipEvent_t) { return done(g_idle ? hipSuccess : hipErrorNotReady); }
hipError_t hipEventDestroy(hipEvent_t e) {
    delete reinterpret_cast<Event*>(e);
    return hipSuccess;
}
hipError_t hipDeviceSynchronize(void) { return hipSuccess; }
}

namespace {
#define CHECK(cond)                                                                      \
    do {                                                                                 \
        if (!(cond)) {                                                                   \
            std::fprintf(stderr, "CHECK failed %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            std::exit(1);                                                                \
        }                                                                                \
    } while (0)

constexpr size_t kBytes = 1 << 20;
hipStream_t stream(int k) { return reinterpret_cast<hipStream_t>(uintptr_t(0x10000 + 16 * k)); }
bool live(void* p) {
    std::lock_guard<std::mutex> lock(g_mu);
    return g_live.count(p) != 0;
}
void* touch(hipStream_t s) {
    const tq::WorkspaceTurn turn(s);
    return tq::workspace(s, kBytes);
}
void nap(int ms) { std::this_thread::sleep_for(std::chrono::milliseconds(ms)); }

// Takes a turn and its buffer, then uses the buffer a while later.
struct Holder {
    std::atomic<bool> has{false};
    std::thread thread;
    explicit Holder(hipStream_t s) {
        thread = std::thread([this, s] {
            const tq::WorkspaceTurn turn(s);
            char* p = static_cast<char*>(tq::workspace(s, kBytes));
            has = true;
            nap(300);
            std::memset(p, 1, kBytes);
        });
        while (!has) nap(1);
    }
    ~Holder() { thread.join(); }
};

void release() {
    for (int k = 0; k < 4; ++k) {
        touch(stream(9));
        Holder holder(stream(k));
        tq::release_workspaces();
    }
    CHECK(g_live.empty());
    touch(stream(1));
    CHECK(g_live.size() == 1);
}

// Streams whose turns do not wait for that of s.
std::vector<hipStream_t> others(hipStream_t s, int n) {
    std::vector<std::atomic<bool>> got(n + 40);
    std::vector<std::thread> all;
    std::vector<hipStream_t> out;
    {
        const tq::WorkspaceTurn turn(s);
        for (int k = 0; k < n + 40; ++k)
            all.emplace_back([&got, k] {
                const tq::WorkspaceTurn t(stream(1000 + k));
                got[k] = true;
            });
        const auto count = [&] {
            int c = 0;
            for (auto& g : got) c += g ? 1 : 0;
            return c;
        };
        for (int ms = 0; ms < 20000 && count() < n; ++ms) nap(1);
        for (int k = 0; k < n + 40 && (int)out.size() < n; ++k)
            if (got[k]) out.push_back(stream(1000 + k));
    }
    for (auto& t : all) t.join();
    CHECK((int)out.size() == n);
    return out;
}

void evict() {
    const std::vector<hipStream_t> rest = others(stream(0), 100);
    Holder holder(stream(0));
    for (hipStream_t s : rest) touch(s);  // (64 are cached: the holder's is the oldest)
    CHECK(holder.has && g_live.size() == 64);
}

void threads() {
    void *mine = touch(hipStreamPerThread), *other = nullptr;
    std::atomic<bool> used{false}, over{false};
    g_idle = false;
    std::thread t([&] {
        t_has_work = true;
        other = touch(hipStreamPerThread);
        used = true;
        while (!over) nap(1);
    });
    while (!used) nap(1);
    CHECK(mine != other);
    CHECK(touch(hipStreamPerThread) == mine);
    // Evicted from another thread, a buffer waits for its own thread's work.
    for (int k = 0; k < 100; ++k) touch(stream(k));
    CHECK(live(other));
    over = true;
    t.join();
    for (int k = 0; k < 100; ++k) touch(stream(200 + k));
    CHECK(live(other));
    g_idle = true;
    for (int k = 0; k < 100; ++k) touch(stream(400 + k));
    CHECK(!live(other) && !live(mine));
    CHECK(g_live.size() == 64);
    tq::release_workspaces();
    CHECK(g_live.empty());
}
}  // namespace

int main(int argc, char** argv) {
    const std::string what = argc > 1 ? argv[1] : "";
    if (what == "release") release();
    else if (what == "evict") evict();
    else if (what == "threads") threads();
    else return 2;
    std::puts("ok");
    return 0;
}
