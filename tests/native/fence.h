// A copy of x whose end is the end of a page, with a page behind it that no access may touch.
#pragma once
#include <sys/mman.h>
#include <unistd.h>

#include <cstring>
#include <vector>

template <typename T>
static T *fenced(const std::vector<T> &x) {
  const size_t page = static_cast<size_t>(sysconf(_SC_PAGESIZE)), bytes = x.size() * sizeof(T);
  const size_t room = (bytes + page - 1) / page * page;
  char *base = static_cast<char *>(
      mmap(nullptr, room + page, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0));
  if (base == MAP_FAILED || mprotect(base + room, page, PROT_NONE) != 0) return nullptr;
  char *at = base + room - bytes;
  std::memcpy(at, x.data(), bytes);
  return reinterpret_cast<T *>(at);
}
