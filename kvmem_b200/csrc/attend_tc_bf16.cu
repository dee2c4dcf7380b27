#include "attend_tc_launch.cuh"

namespace kvmb {
template int launch_attend_tc_t<true>(kvm_ctx*, const AttendTcMaps&, const AttendParams&, uint32_t, int, bool, uint32_t, cudaStream_t);
}  // namespace kvmb
