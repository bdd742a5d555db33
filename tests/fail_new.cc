// fail_new.cc -- operator new that fails once, at the call asked for; preloaded by tests of what the library does
// when host memory runs out.  Allocations of the stand-in runtime (libfake_hip.so) are neither counted nor failed.
#include <dlfcn.h>
#include <stddef.h>
#include <stdlib.h>
#include <string.h>

#include <new>

namespace {
thread_local long left = 0;
thread_local int failed = 0;
void* allocate(size_t n, void* caller) {
  Dl_info from;
  if (left > 0 && !(dladdr(caller, &from) && strstr(from.dli_fname, "fake_hip")) && --left == 0) {
    failed = 1;
    return nullptr;
  }
  return malloc(n ? n : 1);
}
}  // namespace

extern "C" {
// The n-th allocation of this thread from now on fails (0: none does).
void fail_new_at(long n) {
  left = n;
  failed = 0;
}
// Whether it has.
int fail_new_did() { return failed; }
}

void* operator new(size_t n, const std::nothrow_t&) noexcept { return allocate(n, __builtin_return_address(0)); }
void* operator new(size_t n) {
  void* p = allocate(n, __builtin_return_address(0));
  if (!p) throw std::bad_alloc();
  return p;
}
void* operator new[](size_t n) {
  void* p = allocate(n, __builtin_return_address(0));
  if (!p) throw std::bad_alloc();
  return p;
}
void operator delete(void* p) noexcept { free(p); }
void operator delete(void* p, size_t) noexcept { free(p); }
void operator delete[](void* p) noexcept { free(p); }
void operator delete[](void* p, size_t) noexcept { free(p); }
