// rf_verify.h - what the drafted-token verification operators share: argument
// checks of a K/V cache view and the device word their kernels report into.
#pragma once
#include "rf_common.h"

namespace rf {

// Bits of the word rf_verify_error_word reads.
constexpr unsigned kVerifyTimeout = 1u, kVerifyRange = 2u;

inline uint32_t act_bytes(int act_type) {
  return act_type == RF_ACT_F32 ? 4 : act_type == RF_ACT_F16 || act_type == RF_ACT_BF16 ? 2 : 0;
}
inline bool aligned_to(const void* p, uint32_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// RF_OK, or RF_EINVAL / RF_EUNSUPPORTED with a message naming what is wrong with the view.
int check_kv_view(const rf_kv_view* c);
// Address of the current device's error word (looked up in the current context on every call).
int verify_error_ptr(unsigned** out);

}  // namespace rf
