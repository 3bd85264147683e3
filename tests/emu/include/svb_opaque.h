// TEST INFRASTRUCTURE ONLY: lane-emulator stand-in for csrc/svb_opaque.h.
#pragma once
static inline void svb_opaque(unsigned&) {}
static inline void svb_opaque(float&) {}
static inline void svb_opaque_uniform(long long&) {}
static inline void svb_opaque(long long&) {}
