// Host build of dimo_amd/csrc/{experts,grouped}.hip (routing, grouping, grouped products) on the SIMT emulation shim.
// TEST INFRASTRUCTURE ONLY: the expert entry points are exported as they are and take host
// pointers here.
#include "common.hpp"

namespace dimo {
void set_last_error(hipError_t, const char *) {}
ScopedTimer::ScopedTimer(int id, hipStream_t s) : id_(id), stream_(s), a_(nullptr), b_(nullptr) {}
ScopedTimer::~ScopedTimer() {}
}  // namespace dimo
