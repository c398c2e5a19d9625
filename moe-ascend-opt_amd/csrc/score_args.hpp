// score_args.hpp -- argument rules of the score router, for the device and the
// host entry points.  Plain C++.
#pragma once
#include <stdint.h>

namespace mimoe {

// What is wrong with a score router's arguments, or null.
inline const char* score_args_error(int64_t T, int64_t E, int64_t K, int score, int64_t n_group, int64_t topk_group,
                                    int64_t group_top) {
  if (T < 0 || T > ((int64_t)1 << 24)) return "T must be in [0, 2^24]";
  if (E < 1 || E > 512) return "E must be in [1, 512]";
  if (score != 0 && score != 1) return "score must be 0 (softmax) or 1 (sigmoid)";
  if (n_group < 1 || n_group > 64 || E % n_group) return "n_group must be in [1, 64] and divide E";
  if (topk_group < 1 || topk_group > n_group) return "topk_group must be in [1, n_group]";
  if (group_top < 1 || group_top > 2 || (topk_group < n_group && group_top > E / n_group))
    return "group_top must be 1 or 2, and no more than a group holds where groups are dropped";
  if (K < 1 || K > 64 || K > topk_group * (E / n_group)) return "top_k must be in [1, 64] and no more than the chosen groups hold";
  return nullptr;
}

}  // namespace mimoe
