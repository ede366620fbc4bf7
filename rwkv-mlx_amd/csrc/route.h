// Launchers of route.hip; shapes are checked by ops_api.hip.
#pragma once

#include "internal.h"

namespace rwkvmoe {

constexpr int kRouteMaxE = 512, kRouteMaxK = 32, kRouteMaxGroups = 64;

struct Route {
  int rows, E, k, groups, top_groups;
  int dtype;         // of logits and d_logits
  bool sigmoid, top2, renorm;
  float scale;
  long long stride;  // elements between the rows of logits
  const void* logits;
  const float* bias; // or null
  int* inds;         // (rows, k)
  float* gates;      // (rows, k)
  // backward
  const int* inds_in;
  const float* gates_in;
  const float* d_gates;
  void* d_logits;    // (rows, E)
};
hipError_t launch_route(const Route& p, hipStream_t s);
hipError_t launch_route_backward(const Route& p, hipStream_t s);

}  // namespace rwkvmoe
