// Launcher of the one-kernel backward (fa_bwd_fused_kernel.h): softmax_d pass (which also clears the hand-over counters),
// then the kernel.
//
// A workgroup waits for others of its launch, so those have to find a place: one launch at a time on a device.  Two launches' workgroups leave each
// other room (an XCD holds 64, and at most 31 of a launch wait for a pair of which a part has not begun), three do not: each would wait for what the others
// keep out until its polls are used up, and poison its blocks.  A launch therefore waits for the one before it, whatever their streams; under capture, where that
// is not known, the two-kernel backward runs.
#include <mutex>

#include "fa_bwd_fused_kernel.h"

#ifdef FA_FUSED_EXPERIMENTS
#include <cstdio>
#include <cstdlib>
#endif

namespace fa {

namespace {
template <typename T>
hipError_t launch_fused_t(const BwdParams& p0, hipStream_t stream, hipEvent_t ev_start, hipEvent_t ev_stop) {
  BwdParams p = p0;
  const int BH = p.B * p.H;
#ifdef FA_FUSED_EXPERIMENTS
  static const int ring_stride = getenv("FA_RING_STRIDE") ? atoi(getenv("FA_RING_STRIDE")) : 0;
  p.ring_stride = ring_stride;
#endif
  const dim3 gd((p.max_sq + 31) / 32, BH);
  hipLaunchKernelGGL(fused_prepass_kernel<T>, gd, dim3(256), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int grid = tile_grid(false, p.nk_tiles, BH);
  if (ev_start && (e = hipEventRecord(ev_start, stream)) != hipSuccess) return e;
#ifdef FA_FUSED_EXPERIMENTS
  static const int mode = getenv("FA_FUSED_MODE") ? atoi(getenv("FA_FUSED_MODE")) : 0;
  if (mode == 1) hipLaunchKernelGGL((fa_bwd_fused_kernel<T, 64, 1>), dim3(grid), dim3(256), 0, stream, p);
  else if (mode == 2) hipLaunchKernelGGL((fa_bwd_fused_kernel<T, 64, 2>), dim3(grid), dim3(256), 0, stream, p);
  else if (mode == 3) hipLaunchKernelGGL((fa_bwd_fused_kernel<T, 64, 3>), dim3(grid), dim3(256), 0, stream, p);
  else if (mode == 4) hipLaunchKernelGGL((fa_bwd_fused_kernel<T, 64, 4>), dim3(grid), dim3(256), 0, stream, p);

  else
#endif
  hipLaunchKernelGGL((fa_bwd_fused_kernel<T, 64, 0>), dim3(grid), dim3(256), 0, stream, p);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (ev_stop && (e = hipEventRecord(ev_stop, stream)) != hipSuccess) return e;
  return hipSuccess;
}
}  // namespace

namespace {
constexpr int kMostDevices = 64;
std::mutex g_in_turn;
hipEvent_t g_last_done[kMostDevices];  // of a device's last launch; created with its first one and kept
}  // namespace

bool fused_bwd_possible(hipStream_t stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream, &status) == hipSuccess) return status == hipStreamCaptureStatusNone;
  (void)hipGetLastError();
  return false;
}

hipError_t launch_bwd_fused(const BwdParams& p, int dtype, hipStream_t stream, hipEvent_t ev_start, hipEvent_t ev_stop) {
  if (p.B * p.H == 0) return hipSuccess;
  int device = 0;
  hipError_t e = hipGetDevice(&device);
  if (e != hipSuccess) return e;
  if (device < 0 || device >= kMostDevices) return hipErrorInvalidDevice;
  const std::lock_guard<std::mutex> lock(g_in_turn);
  hipEvent_t& done = g_last_done[device];
  if (done) e = hipStreamWaitEvent(stream, done, 0);
  else e = hipEventCreateWithFlags(&done, hipEventDisableTiming);
  if (e != hipSuccess) return e;
  e = dtype == 0 ? launch_fused_t<_Float16>(p, stream, ev_start, ev_stop) : launch_fused_t<__bf16>(p, stream, ev_start, ev_stop);
  return e != hipSuccess ? e : hipEventRecord(done, stream);
}

}  // namespace fa
