// What a plan's kernels keep in shared memory, in 32-bit words, for B requests on a state of R rows:
//   len [B] lengths before | first [B + 1] prefix sums of the tokens | moved [B + 1] prefix sums of the pages that move
// A bit for each row (named by a request yet?) lies over first and moved, from the same place on, until the sums are formed; a state may have many more rows
// than a call has requests, so the larger of the two is what a launch allocates.  (4000 requests on 131072 rows: 48008 bytes.)
#pragma once

namespace mb200 {

constexpr int plan_first_at(int B) { return B; }
constexpr int plan_moved_at(int B) { return 2 * B + 1; }
constexpr int plan_named_at(int B) { return plan_first_at(B); }
constexpr int plan_named_words(int R) { return (R + 31) / 32; }
constexpr int plan_words(int B, int R) {
  return plan_moved_at(B) + B + 1 > plan_named_at(B) + plan_named_words(R) ? plan_moved_at(B) + B + 1 : plan_named_at(B) + plan_named_words(R);
}

}  // namespace mb200
