// What the files of the vocabulary head's losses share: the launches of its products (linear_loss_products.hip and linear_loss_few.hip), made by linear_loss.hip.
#pragma once
#include "tf24_common.hpp"

namespace tf24 {

struct HeadProduct;
struct HeadResult;

// smooth: with a sum of the logits (STATS), less a level (SLOPE), less what all rows have in common (INPUT, WEIGHT); wide: float32 results (WEIGHT)
int launch_head_product(int kind, int dtype, bool smooth, bool wide, const HeadProduct& p, const HeadResult& r, void* stream);

// the forward product of up to kFewTokens tokens (linear_loss_few.hip), operands as they lie: slabs of kFewSlab words, bias as it is
constexpr int kFewTokens = 64, kFewSlab = 64;
struct FewTokens {
  int tokens, filled;
  const int64_t* targets;            // null: which tokens count has been found out already
  int64_t ignore;
  int *count, *row_of, *place_of, *listed;
  float* loss;                       // of tokens that do not count, if there is one of each
};
int launch_few_tokens(int dtype, bool smooth, const FewTokens& which, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t width, const void* bias,
                      int bias_dtype, const HeadResult& r, void* stream);

}  // namespace tf24
