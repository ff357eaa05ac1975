// Fibers, launches and the C entries of the kernels under test; see host_hip.h.  The .hip sources follow as build.py has prepared them.
#include <cstdarg>
#include "host_hip.h"

namespace host {
Fiber fibers[kMaxThreads];
Wave waves[kMaxThreads / kLanes];
int cur, nthreads, bar_count, bar_gen, bar_alive;
dim3 block_idx, block_dim, grid_dim;
char lds_anchor;
static char* stacks;
static void* main_sp;
static const std::function<void()>* body;
extern "C" void host_switch(void** save, void* to);
asm(".text\n.globl host_switch\nhost_switch:\n"
    "pushq %rbp\npushq %rbx\npushq %r12\npushq %r13\npushq %r14\npushq %r15\n"
    "movq %rsp,(%rdi)\nmovq %rsi,%rsp\n"
    "popq %r15\npopq %r14\npopq %r13\npopq %r12\npopq %rbx\npopq %rbp\nret\n");

static int next_live(int i) {
  for (int n = 0; n < nthreads; ++n) { i = i + 1 == nthreads ? 0 : i + 1; if (!fibers[i].done) return i; }
  return -1;
}
void yield() {
  const int from = cur, to = next_live(cur);
  if (to == from) { fprintf(stderr, "host_hip: a collective that not every lane reaches\n"); abort(); }
  cur = to;
  host_switch(&fibers[from].sp, fibers[to].sp);
}
static void entry() {
  (*body)();
  Fiber& f = fibers[cur];
  f.done = true;
  // lanes that have ended take no part in what the others wait for
  Wave& w = waves[f.wave];
  if (--w.alive > 0 && w.count == w.alive) { fprintf(stderr, "host_hip: a lane ended inside its wave's collective\n"); abort(); }
  if (--bar_alive > 0 && bar_count == bar_alive) { bar_count = 0; ++bar_gen; }
  const int from = cur, to = next_live(cur);
  void* sp = to < 0 ? main_sp : fibers[to].sp;
  if (to >= 0) cur = to;
  host_switch(&fibers[from].sp, sp);
}
void launch(dim3 grid, dim3 block, const std::function<void()>& f) {
  if (stacks == nullptr) stacks = (char*)aligned_alloc(4096, (size_t)kMaxThreads * kStack);
  nthreads = (int)(block.x * block.y * block.z);
  if (nthreads < 1 || nthreads > kMaxThreads || (uint64_t)grid.x * block.x >= (1ull << 32) || grid.y > 65535 || grid.x < 1 || grid.y < 1) { fprintf(stderr, "host_hip: launch outside the limits\n"); abort(); }
  body = &f;
  block_dim = block; grid_dim = grid;
  for (unsigned y = 0; y < grid.y; ++y)
    for (unsigned x = 0; x < grid.x; ++x) {
      block_idx = dim3(x, y, 0);
      bar_count = bar_gen = 0; bar_alive = nthreads;
      for (int i = 0; i < (nthreads + kLanes - 1) / kLanes; ++i) { waves[i].count = waves[i].gen = 0; waves[i].alive = std::min(kLanes, nthreads - i * kLanes); }
      for (int i = 0; i < nthreads; ++i) {
        Fiber& b = fibers[i];
        b.tid = dim3(i, 0, 0); b.wave = i / kLanes; b.lane = i % kLanes; b.done = false;
        void** sp = (void**)(stacks + (size_t)(i + 1) * kStack) - 2;
        *--sp = nullptr;
        *--sp = (void*)entry;
        for (int r = 0; r < 6; ++r) *--sp = nullptr;
        b.sp = sp;
      }
      cur = 0;
      host_switch(&main_sp, fibers[0].sp);
    }
}
}  // namespace host

static char g_err[512];
namespace ms {
void set_error(const char* fmt, ...) { va_list ap; va_start(ap, fmt); vsnprintf(g_err, sizeof(g_err), fmt, ap); va_end(ap); }
int num_cus() { return 256; }
}  // namespace ms
extern "C" const char* host_last_error() { return g_err; }
