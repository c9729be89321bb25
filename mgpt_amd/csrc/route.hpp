// route.hpp -- what route.hip shares with the layer (moe_capi.hip).
#pragma once

#include "../../include/mgpt_moe.h"
#include "common.hpp"

namespace mgpt {

constexpr int kRouteRenorm = 1;
constexpr int kRouteDrop = (int)0x80000000;   // what takes no part has the id -1, instead of the lowest ids left

struct RouteArgs {
  const void* logits;    // [N][E]
  const float* bias;     // [E] or null
  int32_t* idx;          // [N][k]
  float* weights;        // [N][k]
  int32_t* counts;       // [E], added to, or null
  // backward
  const int32_t* bidx;
  const float *bw, *dw, *dscore;   // dscore [E] or null
  void* dlogits;
  int N, E, k, G, S, top_groups, best;   // S = E / G
  float scale;
  int vec;
  int how;               // one register: kRouteRenorm, kRouteDrop
};

int check_route(const mgpt_route_config* cfg, int N);   // a status
RouteArgs route_args(const mgpt_route_config* cfg, const void* logits, const void* dlogits, int N);
hipError_t launch_route(const mgpt_route_config* cfg, const RouteArgs& g, bool backward, hipStream_t st);
// A routing for the layer: ids outside 0 .. E - 1 and those of weight 0 become -1 with weight 0 (from -> idx, w; null:
// idx as it is), and hist[e][block of 64 tokens], where not null, as the permute reads it, without the ids -1.
hipError_t launch_route_take(const int32_t* from, const float* from_w, int N, int E, int k, int32_t* idx, float* w,
                             int32_t* hist, hipStream_t st);
// dscore[e] = alpha E counts[e] / N^2: the balance loss' gradient for every token's score.
hipError_t launch_route_dscore(const int32_t* counts, int E, int N, float alpha, float* dscore, hipStream_t st);

}  // namespace mgpt
