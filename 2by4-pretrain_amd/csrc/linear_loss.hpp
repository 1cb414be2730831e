// What the files of the vocabulary head's losses share: the launches of its products (linear_loss_products.hip), made by linear_loss.hip.
#pragma once
#include "tf24_common.hpp"

namespace tf24 {

struct HeadProduct;
struct HeadResult;

// smooth: with a sum of the logits (STATS) or a level that is subtracted (SLOPE); wide: float32 results (WEIGHT)
int launch_head_product(int kind, int dtype, bool smooth, bool wide, const HeadProduct& p, const HeadResult& r, void* stream);

}  // namespace tf24
