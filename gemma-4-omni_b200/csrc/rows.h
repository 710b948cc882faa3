// Whether two strided tensors share memory (host code).
#pragma once
#include <algorithm>
#include <cstdint>

namespace lb {

// [tokens][heads][width]: steps and the width in bytes, the last dimension contiguous.
struct Rows {
  const void* at;
  int64_t token;
  int64_t head;
  int64_t tokens, heads, width;
};

// Exact for equal steps between tokens.  Others that lie in one another's gaps, and those of more than 2^20 pairs of heads that are not
// simply beside one another, count as sharing memory.
inline bool rows_meet(const Rows& a, const Rows& b) {
  if (a.tokens < 1 || a.heads < 1 || b.tokens < 1 || b.heads < 1) return false;
  const int64_t span_a = (a.heads - 1) * a.head + a.width, span_b = (b.heads - 1) * b.head + b.width;
  const int64_t more_a = a.tokens - 1, more_b = b.tokens - 1;
  const int64_t far = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.at) - reinterpret_cast<uintptr_t>(a.at));
  if (far >= (more_a ? more_a * a.token : 0) + span_a || -far >= (more_b ? more_b * b.token : 0) + span_b) return false;
  if (more_a != more_b || (more_a && a.token != b.token)) return true;
  const int64_t token = more_a ? a.token : 0;
  if (token > 0) {
    const int64_t left = (far % token + token) % token;
    if (left >= span_a && left + span_b <= token) return false;  // beside one another in each token
  }
  if (a.heads * b.heads > 1 << 20) return true;
  for (int64_t i = 0; i < a.heads; ++i)
    for (int64_t j = 0; j < b.heads; ++j) {
      // b's head begins d behind a's, and d + m * token behind that of a token m before; the last that begins before a's head ends
      int64_t d = far + j * b.head - i * a.head;
      if (token > 0) {
        const int64_t room = a.width - 1 - d, m = room >= 0 ? room / token : -((-room + token - 1) / token);
        if (m < -more_a) continue;
        d += std::min(m, more_a) * token;
      }
      if (-b.width < d && d < a.width) return true;
    }
  return false;
}

}  // namespace lb
