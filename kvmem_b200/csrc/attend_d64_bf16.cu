#include "attend_launch.cuh"

namespace kvmb {
template int launch_attend_t<64, true>(kvm_ctx*, const AttendParams&, int, bool, int, cudaStream_t);
}  // namespace kvmb
