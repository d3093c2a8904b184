// The lanes of hip/hip_runtime.h as fibers, memory between guard pages, and what the library's sources ask of each other.
#include <hip/hip_runtime.h>

#include <signal.h>
#include <sys/mman.h>
#include <ucontext.h>
#include <unistd.h>

#include <cstdarg>
#include <vector>

LaneIndex threadIdx, blockIdx;

namespace trace {
alignas(64) char lds[160 * 1024];                      // of the workgroup that runs
static char error_text[512];
void set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(error_text, sizeof error_text, fmt, ap);
  va_end(ap);
}
}  // namespace trace

namespace lanes {
namespace {
constexpr size_t STACK = 256 * 1024;
struct Fiber {
  ucontext_t at;
  bool done;
};
struct Wave {
  alignas(64) char slots[2][64 * 128];
  unsigned turn, here;
};
std::vector<Fiber> fibers;
std::vector<Wave> waves;
ucontext_t scheduler;
unsigned threads, barrier_turn, barrier_here, steps;
void (*body)(const void*);
const void* body_args;

void wait_until_turns(const unsigned& turn, unsigned was) {
  const unsigned me = threadIdx.x;
  while (turn == was) swapcontext(&fibers[me].at, &scheduler);
}
void start() {
  const unsigned me = threadIdx.x;
  body(body_args);
  fibers[me].done = true;
  ++steps;
  swapcontext(&fibers[me].at, &scheduler);
}
}  // namespace

const char* wave_all(const void* in, size_t bytes) {
  Wave& w = waves[threadIdx.x / 64];
  const unsigned was = w.turn;
  char* all = w.slots[was & 1];                        // the next operation's go to the other half
  memcpy(all + 128 * (threadIdx.x & 63), in, bytes);
  ++steps;
  if (++w.here == 64) {
    w.here = 0;
    ++w.turn;
  }
  wait_until_turns(w.turn, was);
  return all;
}

void workgroup_barrier() {
  const unsigned was = barrier_turn;
  ++steps;
  if (++barrier_here == threads) {
    barrier_here = 0;
    ++barrier_turn;
  }
  wait_until_turns(barrier_turn, was);
}

void run(unsigned grid, unsigned block, size_t lds_bytes, void (*what)(const void*), const void* args) {
  static std::vector<char> stacks;
  if (lds_bytes > sizeof trace::lds || block % 64) abort();
  stacks.resize(block * STACK);
  threads = block;
  body = what;
  body_args = args;
  for (blockIdx.x = 0; blockIdx.x < grid; ++blockIdx.x) {
    memset(trace::lds, 0xff, sizeof trace::lds);       // NaN: nothing may count on what was there
    fibers.assign(block, Fiber{});
    waves.assign(block / 64, Wave{});
    barrier_turn = barrier_here = 0;
    for (unsigned t = 0; t < block; ++t) {
      getcontext(&fibers[t].at);
      fibers[t].at.uc_stack.ss_sp = stacks.data() + t * STACK;
      fibers[t].at.uc_stack.ss_size = STACK;
      makecontext(&fibers[t].at, start, 0);
    }
    for (unsigned left = block; left;) {
      const unsigned before = steps;
      left = 0;
      for (unsigned t = 0; t < block; ++t) {
        if (fibers[t].done) continue;
        threadIdx.x = t;
        swapcontext(&scheduler, &fibers[t].at);
        left += !fibers[t].done;
      }
      if (left && steps == before) {
        fprintf(stderr, "workgroup %u: lanes wait for others that do not come\n", blockIdx.x);
        _exit(4);
      }
    }
  }
}
}  // namespace lanes

extern "C" const char* lanes_error() { return trace::error_text; }

// `bytes` of memory that end (front: begin) at 256 MB which may not be touched.  Never given back.
extern "C" void* lanes_alloc(size_t bytes, int front) {
  const size_t page = 4096, room = (bytes + page - 1) / page * page, guard = (size_t)256 << 20;
  char* p = static_cast<char*>(mmap(nullptr, room + 2 * guard, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0));
  if (p == MAP_FAILED || (room && mprotect(p + guard, room, PROT_READ | PROT_WRITE))) abort();
  return front ? p + guard : p + guard + room - bytes;
}

static void outside(int, siginfo_t* info, void*) {
  static const char text[] = "access outside of the tensors\n";
  if (write(2, text, sizeof text - 1)) _exit(3);
}
extern "C" void lanes_watch() {
  static char stack[64 * 1024];
  stack_t s{};
  s.ss_sp = stack;
  s.ss_size = sizeof stack;
  sigaltstack(&s, nullptr);
  struct sigaction a {};
  a.sa_sigaction = outside;
  a.sa_flags = SA_SIGINFO | SA_ONSTACK;
  sigaction(SIGSEGV, &a, nullptr);
  sigaction(SIGBUS, &a, nullptr);
}
