// What the translation units of the C ABI share: the error message of the calling thread, argument checks, and the
// library-wide state that api.hip keeps (environment switches, the XCD probe, profiling events).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/g4b_attn.h"

namespace g4b::api {

int fail(int code, const char* fmt, ...);  // sets g4b_last_error() and returns code

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool dtype_ok(int dt) { return dt == G4B_DT_F16 || dt == G4B_DT_BF16 || dt == G4B_DT_F32; }
inline int dtype_bytes(int dt) { return dt == G4B_DT_F32 ? 4 : 2; }

// Partial slots of a decode-shaped launch over nw workers: the segments of workers and pairs form a staircase.
inline uint64_t decode_slots(int B, int G, int nw) { return (uint64_t)nw + (uint64_t)B * G; }
int default_decode_workers(int D);
bool print_plan();
bool xcd_parity(hipStream_t stream);  // workgroup i of a grid runs on an XCD of the parity of i
bool arm_profile();                   // false: the events could not be created
void disarm_profile();

}  // namespace g4b::api
