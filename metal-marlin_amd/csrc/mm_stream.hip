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
