// What the bits of the context's device error word say (hb_check_device).  Plain C++: the message is made on the host.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cstdio>

// Pipeline waits inside the 8-bit products: one bit for the kernels, one for the wait, of which other kernels use the second alone.
enum : uint32_t {
  kErrFp8 = 0x800000u,
  kErrFp8Stage = kErrFp8 | 0x100u,        // a stage of operands to become free
  kErrFp8AccFree = kErrFp8 | 0x200u,      // an accumulator to become free (MMA)
  kErrFp8Loads = kErrFp8 | 0x400u,        // operands to land
  kErrFp8Mma = kErrFp8 | 0x800u,          // the last MMA to end
  kErrFp8Acc = kErrFp8 | 0x1000u,         // an accumulator's sums
  kErrFp8ScaleFree = kErrFp8 | 0x2000u,   // an accumulator to become free (scales)
};

inline void hb_device_error_text(uint32_t v, char* out, size_t n) {
  if (v & kErrFp8)
    snprintf(out, n, "device error word 0x%x (0x800000: a pipeline wait inside an 8-bit product gave up, on 0x100: a free stage, 0x200 or 0x2000: a free accumulator, 0x400: operands, 0x800: the last "
             "MMA, 0x1000: sums; 0x400000: an expert record that is not 16-byte aligned; other bits: an earlier call of another operator)", v);
  else
    snprintf(out, n, "device error word 0x%x (bits 0x1-0x80: a pipeline wait inside a decode or prefill kernel; 0x400-0x2000: the decode layer kernel's tables and grid barrier; "
             "0x40000: rows of another rank did not arrive; 0x80000: partial sums of another rank did not arrive; 0x400000: an expert record that is not 16-byte aligned)", v);
}
