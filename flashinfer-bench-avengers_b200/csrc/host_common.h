// Host helpers shared by the library's entry points (moe_capi.cu has the
// definitions): tensor-map encoding, the device check, small arithmetic.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>

namespace moe {

struct DeviceInfo {
  int checked = 0;
  int ok = 0;
  int sm_count = 0;
};

// MOE_B200_OK and the current device's properties, or the status to return.
int current_device_info(DeviceInfo* out);

// 2-D matrix of `elem_bytes`-wide elements (1 or 2): `rows` rows of `inner`
// elements, `pitch` bytes apart; tiles of box_rows x box_inner elements land
// in shared memory with the 128-byte swizzle, or as plain rows with
// `swizzle` false. Elements outside the matrix read as zero.
bool encode_2d(CUtensorMap* m, const void* base, int elem_bytes, uint64_t inner, uint64_t rows, uint64_t pitch,
               uint32_t box_inner, uint32_t box_rows, bool swizzle = true);

// Devices a per-device setting has been made on (a kernel's shared-memory
// limit): made once, remembered per device.
class OncePerDevice {
 public:
  template <typename F>
  bool operator()(F&& set) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    const uint64_t bit = uint64_t(1) << dev;
    if (done_.load(std::memory_order_acquire) & bit) return true;
    if (!set()) return false;
    done_.fetch_or(bit, std::memory_order_release);
    return true;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

inline int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace moe
