// main() of a kernel on the CPU: <grid> <order> {<file> <bytes> <r|w>} for each pointer of its Args.
// Buffers are read from the files and, with w, written back. order 0 runs the workgroups one behind the
// other, 1 backwards, another number shuffles them by it.
namespace wh {

struct Buffer { char* at; size_t bytes; const char* file; bool back; };
static std::vector<Buffer> buffers;
static const size_t kPage = 4096, kStack = 1 << 16;
static Args args;

// the bytes end where a page that cannot be touched begins; with `low` in the first 4 GiB
static char* guarded(size_t bytes, bool low = false) {
  const size_t size = (bytes + kPage - 1) / kPage * kPage;
  char* p = (char*)mmap(0, size + 2 * kPage, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS | (low ? MAP_32BIT : 0), -1, 0);
  if (p == (char*)MAP_FAILED) stop("no memory");
  mprotect(p, kPage, PROT_NONE);
  mprotect(p + kPage + size, kPage, PROT_NONE);
  memset(p + kPage, 0xFF, size);
  return p + kPage + size - bytes;
}
static void fault(int sig, siginfo_t* si, void*) {
  const char* p = (const char*)si->si_addr;
  fprintf(stderr, "workgroup %u thread %u: signal %d at %p", block.x, me ? me->thread.x : 0, sig, (void*)p);
  for (size_t i = 0; i < buffers.size() && sig == SIGSEGV; i++)
    if (p >= buffers[i].at - 2 * kPage && p < buffers[i].at + buffers[i].bytes + 2 * kPage)
      fprintf(stderr, ", operand %zu at byte %td of %zu", i, p - buffers[i].at, buffers[i].bytes);
  fprintf(stderr, "\n");
  _exit(4);
}
static void lane_main() {
  KERNEL(args);
  if (!me->under_way.empty()) stop("ends with loads into LDS under way");
  me->done = true;
  live--;
  progress++;
  if (live && at_barrier == live) {     // a barrier waits for the waves that have not ended
    at_barrier = 0;
    barrier_gen++;
  }
  for (;;) yield();
}
static void workgroup(unsigned b, char* stacks) {
  block.x = b;
  live = 256, at_barrier = 0;
  for (auto& w : waves) w.count = 0;
  for (unsigned t = 0; t < 256; t++) {
    Lane& l = lanes[t];
    l.thread.x = t, l.done = false, l.under_way.clear();
    void** sp = (void**)(stacks + (t + 1) * kStack);
    *--sp = 0;                          // what lane_main would return to
    *--sp = (void*)lane_main;
    for (int i = 0; i < 6; i++) *--sp = 0;
    l.sp = sp;
  }
  while (live) {
    const unsigned long long before = progress;
    for (auto& l : lanes)
      if (!l.done) {
        me = &l;
        wh_swap(&scheduler, l.sp);
      }
    if (progress == before && live) stop("some lanes wait for others that never come");
  }
}

}  // namespace wh

int main(int argc, char** argv) {
  using namespace wh;
  grid.x = (unsigned)strtoul(argv[1], 0, 10);
  const unsigned order = (unsigned)strtoul(argv[2], 0, 10);
  std::vector<void*> at;
  for (int i = 3; i + 2 < argc; i += 3) {
    Buffer b{0, strtoul(argv[i + 1], 0, 10), argv[i], argv[i + 2][0] == 'w'};
    b.at = guarded(b.bytes);
    FILE* f = fopen(b.file, "rb");
    if (!f || fread(b.at, 1, b.bytes, f) != b.bytes) stop("cannot read an operand");
    fclose(f);
    buffers.push_back(b);
    at.push_back(b.at);
  }
  if (at.size() * sizeof(void*) != sizeof(Args)) stop("the number of operands is not the kernel's");
  memcpy((void*)&args, at.data(), sizeof(Args));
  RING
  static char other[1 << 16];
  stack_t alt{};
  alt.ss_sp = other, alt.ss_size = sizeof other;
  sigaltstack(&alt, 0);
  struct sigaction sa{};
  sa.sa_sigaction = fault, sa.sa_flags = SA_SIGINFO | SA_ONSTACK;
  for (int s : {SIGSEGV, SIGBUS, SIGILL, SIGFPE, SIGTRAP}) sigaction(s, &sa, 0);
  char* stacks = (char*)mmap(0, 256 * kStack, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
  std::vector<unsigned> turn(grid.x);
  for (unsigned i = 0; i < grid.x; i++) turn[i] = order == 1 ? grid.x - 1 - i : i;
  if (order > 1) {
    unsigned long long x = order;
    for (unsigned i = grid.x; i > 1; i--) {
      x = x * 6364136223846793005ULL + 1442695040888963407ULL;
      std::swap(turn[i - 1], turn[(x >> 33) % i]);
    }
  }
  for (unsigned b : turn) workgroup(b, stacks);
  for (auto& b : buffers)
    if (b.back) {
      FILE* f = fopen(b.file, "wb");
      if (!f || fwrite(b.at, 1, b.bytes, f) != b.bytes) return 5;
      fclose(f);
    }
  return 0;
}
