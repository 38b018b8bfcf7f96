// The routing kernels (route.cuh) for 257 to 1024 experts, in a translation
// unit of their own so that the two halves compile at once.
#include "route.cuh"

namespace nvfp4 {
int launch_route_wide(const void* args, int registers, bool softmax, cudaStream_t stream) {
  const RouteArgs& p = *static_cast<const RouteArgs*>(args);
  return registers <= 16 ? launch_route<16>(p, softmax, stream) : launch_route<32>(p, softmax, stream);
}
}  // namespace nvfp4
