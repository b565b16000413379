// nlg_scope.h -- the library's device for the length of a call.
#pragma once

#include "nlg_internal.h"

// The device the library runs on made the calling thread's for one call.
struct NlgDeviceScope {
  int was = -1;
  bool ok = true;
  NlgDeviceScope() {
    const int want = nlg_device();
    if (hipGetDevice(&was) != hipSuccess) was = -1;
    if (was != want) ok = hipSetDevice(want) == hipSuccess;
    else was = -1;
  }
  ~NlgDeviceScope() {
    if (was >= 0) (void)hipSetDevice(was);
  }
};

// (after the checks of arguments: those need no device)
#define NLG_SCOPE(what)                                       \
  if (nlg_ensure_init()) return NLG_ERR;                      \
  NlgDeviceScope scope_;                                      \
  if (!scope_.ok) return nlg_fail("%s: cannot select the library's device", what)
