// CPU test of the operators' workspaces (csrc/op_workspace.h) against a fake of the CUDA
// calls that they make: which stream waits for which work, what a capture gets, and what
// becomes of the memory. Each fake stream has a number and a list of what was put into it.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <string>
#include <thread>
#include <vector>
#include "op_workspace.h"

namespace {
int g_device = 0;
std::string g_log;                            // calls since the last clear()
std::map<cudaStream_t, unsigned long long> g_id;  // handle -> number
std::set<cudaStream_t> g_capturing;
std::set<void *> g_live;
int g_events = 0, g_fail_record = 0;
uintptr_t g_next = 0x1000;
std::string name(cudaStream_t s) { return std::to_string(g_id.at(s)); }
std::string take_log() {
  std::string l = g_log;
  g_log.clear();
  return l;
}
void check(bool ok, char const *what, int line) {
  if (ok) return;
  std::printf("line %d: %s\n", line, what);
  std::exit(1);
}
#define CHECK(x) check(x, #x, __LINE__)
#define CHECK_LOG(want) \
  do { \
    const std::string got = take_log(); \
    if (got != want) std::printf("got: %s\n", got.c_str()); \
    check(got == want, want, __LINE__); \
  } while (0)
}  // namespace

namespace eir {
int api_set_error(int code, char const *) { return code; }
int api_cuda_fail(cudaError_t, char const *) { return EIR_CUDA_ERROR; }
}  // namespace eir

extern "C" {
cudaError_t cudaGetDevice(int *d) { *d = g_device; return cudaSuccess; }
cudaError_t cudaSetDevice(int d) { g_device = d; return cudaSuccess; }
cudaError_t cudaStreamIsCapturing(cudaStream_t s, cudaStreamCaptureStatus *c) {
  *c = g_capturing.count(s) ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
  return cudaSuccess;
}
cudaError_t cudaStreamGetId(cudaStream_t s, unsigned long long *id) { *id = g_id.at(s); return cudaSuccess; }
cudaError_t cudaMemPoolCreate(cudaMemPool_t *p, cudaMemPoolProps const *props) {
  *p = reinterpret_cast<cudaMemPool_t>((uintptr_t)(1 + props->location.id));
  return cudaSuccess;
}
cudaError_t cudaMemPoolSetAttribute(cudaMemPool_t, cudaMemPoolAttr, void *) { return cudaSuccess; }
cudaError_t cudaMemPoolDestroy(cudaMemPool_t) { return cudaSuccess; }
cudaError_t cudaMallocFromPoolAsync(void **p, size_t, cudaMemPool_t pool, cudaStream_t s) {
  *p = reinterpret_cast<void *>(g_next += 0x1000);
  g_live.insert(*p);
  g_log += "alloc on " + std::to_string((uintptr_t)pool - 1) + " in " + name(s) + "; ";
  return cudaSuccess;
}
cudaError_t cudaFree(void *p) {
  CHECK(g_live.erase(p) == 1);
  g_log += "free on " + std::to_string(g_device) + "; ";
  return cudaSuccess;
}
cudaError_t cudaEventCreateWithFlags(cudaEvent_t *e, unsigned) {
  *e = reinterpret_cast<cudaEvent_t>((uintptr_t)++g_next);
  ++g_events;
  return cudaSuccess;
}
cudaError_t cudaEventDestroy(cudaEvent_t) { --g_events; return cudaSuccess; }
cudaError_t cudaEventSynchronize(cudaEvent_t) { g_log += "host waits; "; return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t s) {
  if (g_fail_record > 0 && --g_fail_record == 0) return cudaErrorUnknown;
  g_log += "record in " + name(s) + "; ";
  return cudaSuccess;
}
cudaError_t cudaStreamWaitEvent(cudaStream_t s, cudaEvent_t, unsigned) { g_log += "wait in " + name(s) + "; "; return cudaSuccess; }
}

namespace {
cudaStream_t stream(uintptr_t handle, unsigned long long id) {
  cudaStream_t s = reinterpret_cast<cudaStream_t>(handle);
  g_id[s] = id;
  return s;
}

void order_over_streams() {
  eir::OpWorkspace w;
  cudaStream_t a = stream(16, 1), b = stream(32, 2);
  void *p = nullptr, *q = nullptr;
  CHECK(w.take(64, a, &p) == 0 && p != nullptr);
  CHECK_LOG("alloc on 0 in 1; record in 1; ");
  // the call fails behind take(): the other stream still comes behind the allocation
  CHECK(w.take(64, b, &q) == 0 && q == p);
  CHECK_LOG("wait in 2; ");
  CHECK(w.used(b, 0) == 0);
  CHECK_LOG("record in 2; ");
  CHECK(w.take(64, b, &q) == 0 && w.used(b, 0) == 0);
  CHECK_LOG("record in 2; ");
  // the handle of b is given to a new stream (or is the per-thread default stream of another thread)
  b = stream(32, 3);
  CHECK(w.take(64, b, &q) == 0 && q == p);
  CHECK_LOG("wait in 3; ");
  CHECK(w.used(b, EIR_CUDA_ERROR) == EIR_CUDA_ERROR);
  CHECK_LOG("record in 3; ");
  g_fail_record = 1;
  CHECK(w.used(a, 0) == EIR_CUDA_ERROR);
  w.release();
  CHECK_LOG("host waits; free on 0; ");
  CHECK(g_live.empty() && g_events == 0);
}

void captures() {
  eir::OpWorkspace w;
  cudaStream_t a = stream(16, 1), b = stream(32, 2);
  void *p = nullptr, *q = nullptr;
  g_capturing.insert(a);
  CHECK(w.take(64, a, &p) == EIR_INVALID_ARGUMENT);
  CHECK_LOG("");
  g_capturing.erase(a);
  CHECK(w.take(64, a, &p) == 0 && w.used(a, 0) == 0);
  take_log();
  g_capturing.insert(b);
  CHECK(w.take(64, b, &q) == 0 && q == p && w.used(b, 0) == 0);
  CHECK_LOG("");
  g_capturing.erase(b);
  w.release();
  take_log();
}

// each device has memory of its own, which stays where a graph may use it until the plan is destroyed
void devices() {
  eir::OpWorkspace w;
  cudaStream_t a = stream(16, 1), b = stream(32, 2);
  void *p = nullptr, *q = nullptr;
  CHECK(w.take(64, a, &p) == 0 && w.used(a, 0) == 0);
  CHECK_LOG("alloc on 0 in 1; record in 1; record in 1; ");
  g_device = 1;
  g_capturing.insert(b);
  CHECK(w.take(64, b, &q) == EIR_INVALID_ARGUMENT);
  g_capturing.erase(b);
  CHECK_LOG("");
  CHECK(w.take(64, b, &q) == 0 && q != p && w.used(b, 0) == 0);
  CHECK_LOG("alloc on 1 in 2; record in 2; record in 2; ");
  CHECK(g_live.count(p) == 1);
  g_device = 0;
  g_capturing.insert(a);
  CHECK(w.take(64, a, &q) == 0 && q == p);
  g_capturing.erase(a);
  CHECK(w.take(64, b, &q) == 0 && q == p);
  CHECK_LOG("wait in 2; ");
  w.release();
  CHECK_LOG("host waits; free on 1; host waits; free on 0; ");
  CHECK(g_device == 0 && g_live.empty() && g_events == 0);
}

// two host threads with a stream each call one plan: no call's take() comes between another's take() and used()
void host_threads() {
  eir::OpWorkspace w;
  cudaStream_t s[2] = {stream(16, 1), stream(32, 2)};
  void *p = nullptr;
  CHECK(w.take(64, s[0], &p) == 0 && w.used(s[0], 0) == 0);
  take_log();
  auto calls = [&](int i) {
    for (int j = 0; j < 2000; ++j) {
      auto held = w.hold();
      void *q = nullptr;
      CHECK(w.take(64, s[i], &q) == 0 && q == p);
      g_log += "launch in " + name(s[i]) + "; ";
      std::this_thread::yield();
      CHECK(w.used(s[i], 0) == 0);
    }
  };
  std::thread t0(calls, 0), t1(calls, 1);
  t0.join();
  t1.join();
  // a launch, its record, and a wait before the next launch where that is on the other stream
  std::string log = take_log(), last = "1";
  for (size_t at = 0; at < log.size();) {
    auto next = [&]() {
      const size_t end = log.find("; ", at);
      std::string word = log.substr(at, end - at);
      at = end + 2;
      return word;
    };
    std::string word = next(), now = word.substr(word.size() - 1);
    if (now != last) {
      CHECK(word == "wait in " + now);
      word = next();
    }
    CHECK(word == "launch in " + now);
    CHECK(next() == "record in " + now);
    last = now;
  }
  w.release();
  take_log();
}
}  // namespace

int main() {
  order_over_streams();
  captures();
  devices();
  host_threads();
  std::printf("ok\n");
  return 0;
}
