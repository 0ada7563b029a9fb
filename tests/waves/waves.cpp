// waves.cpp -- runs a kernel's workgroups on the CPU, one after the other (see hip/hip_runtime.h).
#include "hip/hip_runtime.h"

#include <sys/mman.h>

#include <cstdarg>

#include "tm_internal.h"

dim3 blockIdx, gridDim, blockDim;
WavesThreadIdx threadIdx;
int waves_item;
int64_t waves_slot[1024];

// Saves this stack's registers and pointer at *from and goes on with the stack at `to`.
extern "C" void waves_switch(void** from, void* to);
asm(R"(
.text
.globl waves_switch
waves_switch:
  push %rbp
  push %rbx
  push %r12
  push %r13
  push %r14
  push %r15
  mov %rsp, (%rdi)
  mov %rsi, %rsp
  pop %r15
  pop %r14
  pop %r13
  pop %r12
  pop %rbx
  pop %rbp
  ret
)");

namespace {

enum State { kRuns, kMeets, kWaits, kDone };
constexpr size_t kStack = 64 << 10;
constexpr int kMost = 1024;
void* scheduler;
void* item[kMost];
State state[kMost];
const std::function<void()>* body;

void leave(State s) {
  const int mine = waves_item;
  state[mine] = s;
  waves_switch(&item[mine], scheduler);
  waves_item = mine;
}

void begin() {
  (*body)();
  leave(kDone);
  std::abort();
}

[[noreturn]] void wrong(const char* name, const char* what) {
  std::printf("%s, workgroup (%u, %u): %s\n", name, blockIdx.x, blockIdx.y, what);
  std::abort();
}

void run_workgroup(int items, const char* name) {
  static char* stacks = static_cast<char*>(
      mmap(nullptr, kStack * kMost, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0));
  if (stacks == MAP_FAILED) wrong(name, "no memory for stacks");
  for (int t = 0; t < items; ++t) {
    void** sp = reinterpret_cast<void**>(stacks + kStack * (t + 1));
    *--sp = nullptr;
    *--sp = reinterpret_cast<void*>(begin);
    for (int i = 0; i < 6; ++i) *--sp = nullptr;
    item[t] = sp;
    state[t] = kRuns;
  }
  for (;;) {
    int waiting = 0, done = 0;
    for (int first = 0; first < items; first += 64) {
      for (bool again = true; again;) {  // the wave, up to a barrier or its end
        again = false;
        int meets = 0;
        for (int t = first + 63; t >= first; --t) {
          if (state[t] == kRuns) {
            waves_item = t;
            waves_switch(&scheduler, item[t]);
          }
          meets += state[t] == kMeets;
        }
        if (meets == 64) {
          for (int t = first; t < first + 64; ++t) state[t] = kRuns;
          again = true;
        } else if (meets) {
          wrong(name, "a collective that part of a wave reaches");
        }
      }
      for (int t = first; t < first + 64; ++t) {
        waiting += state[t] == kWaits;
        done += state[t] == kDone;
      }
    }
    if (done == items) return;
    if (waiting + done != items) wrong(name, "stuck");
    for (int t = 0; t < items; ++t)
      if (state[t] == kWaits) state[t] = kRuns;
  }
}

}  // namespace

void waves_meet() { leave(kMeets); }
void waves_barrier() { leave(kWaits); }

void waves_launch(dim3 grid, dim3 block, const std::function<void()>& kernel, const char* name) {
  gridDim = grid;
  blockDim = block;
  body = &kernel;
  if (block.x < 64 || block.x > kMost || block.x % 64) wrong(name, "workgroups are whole waves here");
  for (uint32_t y = 0; y < grid.y; ++y)
    for (uint32_t x = 0; x < grid.x; ++x) {
      blockIdx = dim3(x, y);
      run_workgroup(static_cast<int>(block.x), name);
    }
}

int tm_internal_fail(int code, const char* fmt, ...) {
  va_list args;
  va_start(args, fmt);
  std::vprintf(fmt, args);
  va_end(args);
  std::printf("\n");
  return code;
}
