// What the expanded attention may be asked for beyond causal order.
#pragma once

#include "dsa_common.h"

namespace dsa {

struct ExpandedMore {
  const int* first;     // [Tq]: a query's first key in its sequence; null: 0
  const int* last;      // [Tq]: the key behind its last; null: none
  const float* slopes;  // [H]: of the distance between a query's place and a key's, taken off the score; null: none
  float softcap;        // scores become softcap tanh(s / softcap); 0: as they are
};

}  // namespace dsa
