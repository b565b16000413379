// nlg_scope.h -- what an entry point begins with: its arguments against each other, and the library's device for the
// length of the call.
#pragma once

#include "nlg_internal.h"

// Whether two arrays of na and nb bytes share any (a null one shares none).
static inline bool nlg_overlap(const void *a, uint64_t na, const void *b, uint64_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return a && b && x < y + nb && y < x + na;
}

// Arrays of a call, the inputs first: whether any of the last `outs` (outputs, the workspace) shares bytes with another.
struct NlgSpan {
  const void *p;
  uint64_t n;
};
static inline bool nlg_outputs_overlap(const NlgSpan *a, int n, int outs) {
  for (int o = n - outs; o < n; o++)
    for (int i = 0; i < n; i++)
      if ((i < n - outs || i > o) && nlg_overlap(a[o].p, a[o].n, a[i].p, a[i].n)) return true;
  return false;
}

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
