// A workgroup's threads on the CPU: each with a stack of its own, run in turn. The waves go on in random order from stop
// to stop; a wave's threads stop together, at an operation between lanes or at a barrier.
#include <hip/hip_runtime.h>
#include <setjmp.h>
#include <stdio.h>
#include <ucontext.h>

#include <random>
#include <vector>

Dim blockIdx, blockDim;

namespace model {
namespace {

enum State { kRuns, kLanes, kBarrier, kDone };
struct Thread {
  jmp_buf at;
  ucontext_t start;
  State state;
  bool begun;
  uint64_t given;
};
constexpr int kMost = 1024, kStack = 1 << 17;
Thread threads[kMost];
std::vector<char*> stacks;
jmp_buf scheduler;
ucontext_t scheduler_context;
int current;
const std::function<void()>* body;
std::mt19937 chance(1);

void first_step() {
  (*body)();
  threads[current].state = kDone;
  _longjmp(scheduler, 1);
}
// (_setjmp and _longjmp, which leave the signal mask alone, where swapcontext would be two system calls)
void stop(State state) {
  Thread& t = threads[current];
  t.state = state;
  if (!_setjmp(t.at)) _longjmp(scheduler, 1);
}
void run(int i) {
  Thread& t = threads[i];
  current = i, t.state = kRuns;
  if (_setjmp(scheduler)) return;
  if (t.begun) _longjmp(t.at, 1);
  t.begun = true;
  setcontext(&t.start);
}
[[noreturn]] void wrong(const char* what) {
  fprintf(stderr, "workgroup %u, thread %d: %s\n", blockIdx.x, current, what);
  abort();
}

}  // namespace

int thread() { return current; }
void barrier() { stop(kBarrier); }
uint64_t from_lane(uint64_t x, int lane) {
  threads[current].given = x;
  stop(kLanes);
  x = threads[(current & ~63) + lane].given;
  stop(kLanes);
  return x;
}
uint64_t lanes_with(bool x) {
  threads[current].given = x;
  stop(kLanes);
  uint64_t all = 0;
  for (int l = 0; l < 64; ++l) all |= threads[(current & ~63) + l].given << l;
  stop(kLanes);
  return all;
}

void launch(unsigned grid, unsigned block, const std::function<void()>& kernel) {
  if (block % 64 || block > kMost) wrong("not a workgroup of whole waves");
  body = &kernel, blockDim.x = block;
  while (stacks.size() < block) stacks.push_back((char*)malloc(kStack));
  std::vector<unsigned> order(grid);
  for (unsigned i = 0; i < grid; ++i) order[i] = i;
  std::shuffle(order.begin(), order.end(), chance);
  for (unsigned b : order) {
    blockIdx.x = b;
    for (unsigned i = 0; i < block; ++i) {
      Thread& t = threads[i];
      getcontext(&t.start);
      t.start.uc_stack.ss_sp = stacks[i], t.start.uc_stack.ss_size = kStack, t.start.uc_link = nullptr;
      makecontext(&t.start, first_step, 0);
      t.state = kRuns, t.begun = false;
    }
    for (;;) {
      std::vector<int> ready;
      unsigned done = 0, waiting = 0;
      for (unsigned w = 0; w < block; w += 64) {
        bool some = false;
        for (unsigned i = w; i < w + 64; ++i) {
          some |= threads[i].state == kRuns || threads[i].state == kLanes;
          done += threads[i].state == kDone, waiting += threads[i].state == kBarrier;
        }
        if (some) ready.push_back((int)w);
      }
      if (ready.empty()) {
        if (done == block) break;
        if (waiting != block) wrong("a barrier that not all threads reach");
        for (unsigned i = 0; i < block; ++i) threads[i].state = kRuns;
        continue;
      }
      const int w = ready[chance() % ready.size()];
      // those of the wave that are not at an operation between lanes yet go there first
      bool before = false;
      for (int i = w; i < w + 64; ++i) before |= threads[i].state == kRuns;
      for (int i = w; i < w + 64; ++i)
        if (threads[i].state == (before ? kRuns : kLanes)) run(i);
      bool lanes = false, barrier = false;
      for (int i = w; i < w + 64; ++i) lanes |= threads[i].state == kLanes, barrier |= threads[i].state == kBarrier;
      if (lanes && barrier) wrong("lanes of a wave at a barrier, others at an operation between lanes");
    }
  }
}

}  // namespace model

extern "C" __attribute__((visibility("default"))) void model_seed(unsigned seed) { model::chance.seed(seed); }

// (what the compiler calls to round to bf16, to nearest even)
extern "C" __attribute__((visibility("default"))) __bf16 __truncsfbf2(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const uint32_t r = x != x ? u >> 16 | 0x40 : (u + 0x7FFF + (u >> 16 & 1)) >> 16;
  return __builtin_bit_cast(__bf16, (uint16_t)r);
}
