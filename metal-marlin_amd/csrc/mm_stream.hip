// What the host layers ask about a stream: whether it is being captured, and into what.
#include "mm_common.h"
#include "mmfp4.h"

extern "C" unsigned long long mm_capture_id(void* stream) {
  if (stream == nullptr) return 0;   // the default stream cannot be captured
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo((hipStream_t)stream, &status, &id) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return status == hipStreamCaptureStatusNone ? 0 : id;
}

// Also while a stream is being captured: an event recorded before that is no part of it, and the
// relaxed mode is the one that may ask.
extern "C" int mm_event_done(void* event) {
  hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
  if (hipThreadExchangeStreamCaptureMode(&mode) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  const hipError_t e = hipEventQuery((hipEvent_t)event);
  (void)hipThreadExchangeStreamCaptureMode(&mode);
  if (e != hipSuccess) (void)hipGetLastError();
  return e == hipSuccess;
}

// 64 KiB by one wave of every fourth CU, 16 bytes a lane.
constexpr int CC_BYTES = 65536, CC_NT = 64;
__global__ void __launch_bounds__(CC_NT) k_clear_counters(u32x4* ws) {
  ws[blockIdx.x * CC_NT + threadIdx.x] = u32x4{0, 0, 0, 0};
}

extern "C" int mm_clear_counters(void* ws, size_t ws_bytes, void* stream) {
  MM_CHECK_ARG(ws != nullptr && ((uintptr_t)ws & 15) == 0 && ws_bytes >= CC_BYTES,
               "mm_clear_counters: a workspace of %zu bytes must have %d, 16-byte aligned", ws_bytes,
               CC_BYTES);
  hipLaunchKernelGGL(k_clear_counters, dim3(CC_BYTES / (16 * CC_NT)), dim3(CC_NT), 0,
                     (hipStream_t)stream, (u32x4*)ws);
  MM_CHECK_LAUNCH("mm_clear_counters");
  return 0;
}
