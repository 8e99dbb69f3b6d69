// fake_errors.cpp -- the last-error calls of fake_hip.hpp's runtime: nothing is ever pending.
#include <hip/hip_runtime.h>

extern "C" {
hipError_t hipPeekAtLastError() { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
}
