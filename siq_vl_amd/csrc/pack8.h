// Internal interface of the 8-bit activation storage kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace siq {

// Elements that share one scale byte: 32 neighbours in memory order.
constexpr int kPackGroup = 32;

hipError_t launch_pack8(const void* x, int64_t numel, bool f32, bool e4m3, uint8_t* codes, uint8_t* scales,
                        hipStream_t stream);
hipError_t launch_unpack8(const uint8_t* codes, const uint8_t* scales, int64_t numel, bool f32, bool e4m3, void* x,
                          hipStream_t stream);

// Rows of cols elements; *_ld: elements from one row to the next.  Codes and
// scales are those of a contiguous [rows, cols] tensor.
struct SwigluArgs {
  const void* gate;    // forward
  const void* up;
  const void* dh;      // backward
  void* h;             // forward; backward: recomputed, or nullptr
  void* dgate;         // backward
  void* dup;
  uint8_t* gcodes;     // forward: written, or nullptr; backward: read
  uint8_t* gscales;
  uint8_t* ucodes;
  uint8_t* uscales;
  int64_t rows, cols, ld0, ld1;  // of gate and up, or dgate and dup
  bool f32, e4m3;
};
hipError_t launch_swiglu8_fwd(const SwigluArgs& a, hipStream_t stream);
hipError_t launch_swiglu8_bwd(const SwigluArgs& a, hipStream_t stream);

}  // namespace siq
