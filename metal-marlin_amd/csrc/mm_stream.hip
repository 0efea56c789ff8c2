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
