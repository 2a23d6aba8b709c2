// Where a caller's tensor lies, and whether two of them may share an element: plain host arithmetic, without CUDA.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace kb {

// A tensor [n[0]][n[1]][n[2]][width] with strides in elements, 0 or more; the last dimension is contiguous.
struct Box {
  const char* name;
  const void* p;
  int64_t n[3], s[3];
  int64_t width;
  size_t elem;
  bool empty() const { return n[0] == 0 || n[1] == 0 || n[2] == 0 || width == 0; }
  // bytes from the first element to behind the last one
  int64_t bytes() const { return ((n[0] - 1) * s[0] + (n[1] - 1) * s[1] + (n[2] - 1) * s[2] + width) * (int64_t)elem; }
};

// Whether two of its elements may be the same: from the smallest stride up, each has to clear what the dimensions below it span.
inline bool overlapsItself(const Box& b) {
  if(b.empty()) return false;
  int order[3] = {0, 1, 2};
  for(int i = 0; i < 3; i++)
    for(int j = i + 1; j < 3; j++)
      if(b.s[order[j]] < b.s[order[i]]) std::swap(order[i], order[j]);
  int64_t span = b.width;
  for(int i = 0; i < 3; i++) {
    const int d = order[i];
    if(b.n[d] <= 1) continue;
    if(b.s[d] < span) return true;
    span += (b.n[d] - 1) * b.s[d];
  }
  return false;
}

// Whether two tensors may share an element.  Exact enough for parts of one buffer: channel ranges of the same rows do not.
inline bool mayOverlap(Box a, Box b) {
  if(a.empty() || b.empty()) return false;
  const int64_t pa = (int64_t)(uintptr_t)a.p, pb = (int64_t)(uintptr_t)b.p;
  if(pa + a.bytes() <= pb || pb + b.bytes() <= pa) return false;
  // a dimension that repeats (stride 0) reaches nothing new: one of it stands for all
  for(Box* x : {&a, &b})
    for(int i = 0; i < 3; i++)
      if(x->s[i] == 0) x->n[i] = 1;
  // rows of the same stride (tokens, or sequences of one token; batches of whole rows): compare the windows that each takes of a row
  auto rowOf = [](const Box& x) { return (x.n[1] > 1 ? x.s[1] : (x.n[0] > 1 ? x.s[0] : 0)) * (int64_t)x.elem; };
  const int64_t ra = rowOf(a), rb = rowOf(b), row = std::max(ra, rb);
  if(row <= 0 || (ra != 0 && ra != row) || (rb != 0 && rb != row)) return true;
  auto whole = [](const Box& x) { return x.n[0] == 1 || x.n[1] == 1 || x.s[0] % x.s[1] == 0; };
  if(!whole(a) || !whole(b)) return true;
  const int64_t wa = ((a.n[2] - 1) * a.s[2] + a.width) * (int64_t)a.elem, wb = ((b.n[2] - 1) * b.s[2] + b.width) * (int64_t)b.elem;
  if(wa > row || wb > row) return true;
  const int64_t delta = (((pb - pa) % row) + row) % row;
  return delta < wa || delta + wb > row;
}

inline bool sameBox(const Box& a, const Box& b) {
  if(a.p != b.p) return false;
  for(int i = 0; i < 3; i++)
    if(a.n[i] > 1 && a.s[i] != b.s[i]) return false;
  return true;
}

}  // namespace kb
