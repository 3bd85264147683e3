// TEST INFRASTRUCTURE ONLY: lane-emulator stand-in for csrc/svb_opaque.h.
#pragma once
static inline void svb_opaque(unsigned&) {}
