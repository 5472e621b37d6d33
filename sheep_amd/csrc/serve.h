// What the operators of sml-serve.h share on the host (serve.c, rows.c).
#pragma once
#include "ops.h"
#include "sml-serve.h"

static inline int al16(const void * p) { return ((uintptr_t) p & 15u) == 0; }
static inline int ceil_div(int a, int b) { return (int) (((long) a + b - 1) / b); }

// The library's device is current, or the call is refused.
void sv_on_device(void);
// A cache's description checked and as the kernels see it.
void sv_check_pages(const sml_hip_pages * p, sml_kpages * k);
// A kernel's name with the variant of its head size and type.
void sv_name(char * s, size_t n, const char * base, int hd, int type);
