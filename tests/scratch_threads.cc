// Host threads that share the library's scratch memory, without a GPU: runtime.cc linked with the stand-ins below for the
// calls of the CUDA runtime that it makes.  Prints a line for every check that fails; built and run by test_scratch_threads.py.
#include <atomic>
#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <set>
#include <string>
#include <thread>

#include "common.h"

namespace {
std::mutex g_mutex;
std::set<void*> g_live;
std::atomic<bool> g_capturing{false};
int g_failed = 0;

cudaError_t give(void** p, size_t bytes) {
  *p = std::malloc(bytes);
  std::lock_guard<std::mutex> lock(g_mutex);
  g_live.insert(*p);
  return cudaSuccess;
}
cudaError_t take_back(void* p) {
  std::lock_guard<std::mutex> lock(g_mutex);
  g_live.erase(p);  // not returned to malloc: no address comes twice
  return cudaSuccess;
}
bool live(void* p) {
  std::lock_guard<std::mutex> lock(g_mutex);
  return g_live.count(p) != 0;
}
size_t live_count() {
  std::lock_guard<std::mutex> lock(g_mutex);
  return g_live.size();
}
void check(bool ok, const char* what) {
  if (ok) return;
  std::printf("failed: %s\n", what);
  ++g_failed;
}
cudaStream_t stream(int i) { return reinterpret_cast<cudaStream_t>(static_cast<intptr_t>(0x1000 * i)); }

// Takes scratch in another thread while this one holds some; whether it came by before this one let go.
struct Other {
  std::atomic<bool> got{false};
  void* at = nullptr;
  std::thread t;
  Other(cudaStream_t s, size_t bytes)
      : t([this, s, bytes] {
          sptir::CallScratch cs;
          if (sptir::take_scratch(0, s, bytes, 0, &cs) != 0) std::abort();
          at = cs.scratch;
          got = true;
          sptir::return_scratch(cs, s);
        }) {}
  bool within(int ms) {
    for (int i = 0; i < ms && !got; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
    return got;
  }
};
}  // namespace

extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaMalloc(void** p, size_t bytes) { return give(p, bytes); }
cudaError_t cudaFree(void* p) { return take_back(p); }
cudaError_t cudaMallocAsync(void** p, size_t bytes, cudaStream_t) { return give(p, bytes); }
cudaError_t cudaFreeAsync(void* p, cudaStream_t) { return take_back(p); }
cudaError_t cudaMemsetAsync(void*, int, size_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return ""; }
const char* cudaGetErrorName(cudaError_t) { return ""; }
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* s) {
  *s = g_capturing ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
  return cudaSuccess;
}
}

int main() {
  using sptir::CallScratch;
  using sptir::take_scratch;
  // a call that needs more on the same stream, and one that needs as much
  for (size_t bytes : {size_t{64} << 20, size_t{1000}}) {
    Other* other = nullptr;
    {
      CallScratch cs;
      take_scratch(0, stream(1), 1000, 64, &cs);
      other = new Other(stream(1), bytes);
      check(!other->within(100), "a second call on the stream got its scratch before the first call's launches were queued");
      check(live(cs.scratch), "scratch was freed under a call that holds it");
    }
    check(other->within(10000), "the second call never got its scratch");
    other->t.join();
  }
  {  // calls on other streams and calls that are captured wait for nobody
    CallScratch cs;
    take_scratch(0, stream(1), 1000, 0, &cs);
    Other apart(stream(2), 1000);
    check(apart.within(10000) && apart.at != cs.scratch, "a call on another stream waited or shared scratch");
    apart.t.join();
    g_capturing = true;
    Other captured(stream(1), 1000);
    check(captured.within(10000) && captured.at != cs.scratch, "a captured call waited or shared scratch");
    captured.t.join();
    g_capturing = false;
    // the stages of one call
    CallScratch again;
    check(take_scratch(0, stream(1), 1000, 0, &again) == 0 && again.scratch == cs.scratch, "a stage of the same call");
  }
  // one handle, a stream of its own for every thread
  const size_t before = live_count();
  {
    CallScratch cs;
    take_scratch(0, cudaStreamPerThread, 1000, 0, &cs);
    Other own(cudaStreamPerThread, 64 << 20);
    check(own.within(10000), "calls on two threads' own streams waited for each other");
    check(own.at != cs.scratch && live(cs.scratch), "two threads' own streams shared scratch");
    own.t.join();
    check(live_count() == before + 1, "the scratch of a thread's own stream outlived the thread");
  }
  if (g_failed == 0) std::printf("ok\n");
  return g_failed != 0;
}
