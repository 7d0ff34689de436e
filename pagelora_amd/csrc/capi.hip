// Library-wide C entry points: error string, ABI version, which capture a stream is in.
#include "pl_common.h"

extern "C" const char* pl_last_error(void) { return pl::error_buffer(); }

extern "C" int pl_version(void) { return (1 << 16) | 0; }

extern "C" int pl_capture_id(void* stream, unsigned long long* id_h) {
  if (!id_h) return pl::fail(PL_ERR_INVALID, "null pointer argument");
  *id_h = 0;
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  const hipError_t e = hipStreamGetCaptureInfo((hipStream_t)stream, &status, &id);
  if (e != hipSuccess) return pl::fail(PL_ERR_HIP, "hipStreamGetCaptureInfo: %s", hipGetErrorString(e));
  if (status != hipStreamCaptureStatusActive) return pl::fail(PL_ERR_INVALID, "the stream is not captured");
  *id_h = id;
  return pl::ok();
}
