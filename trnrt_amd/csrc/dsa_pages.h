// The caches that one launch of the page operations takes (a kernel argument).
#pragma once

namespace dsa {

constexpr int PG_CACHES = 128;  // 2.6 KB of the 4 KB that a launch's arguments may take

struct PageCaches {
  void* p[PG_CACHES];
  long long page_bytes[PG_CACHES];
  int first[PG_CACHES];  // the first of each cache's pieces within a page's
  int n;
  int pieces;            // of one page of all of them
};

}  // namespace dsa
