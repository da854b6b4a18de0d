// Rows of the linear attention's and the gated norm's calls as their kernels address them.  No HIP: the kernels and the host tests
// compile the same functions.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define POPE_LIN_HD __host__ __device__ __forceinline__
#else
#define POPE_LIN_HD inline
#endif

namespace pope {

// Rows (b, h, n) of `cols` elements.
struct LinRows {
  void* p;
  int64_t s[3];   // elements; s[2] is 0 where there is one row
  int cols;
  int type;       // pope_dtype: 0 fp32, 1 fp16, 2 bf16
  int vec;        // rows of whole, aligned units of 8 elements (outputs of the attention: of 4)
};

POPE_LIN_HD int lin_size(int type) { return type == 0 ? 4 : 2; }
// Bytes from row to row, of rows near each other (chunks of 64 rows at a time, queries' expansion of 256; row strides below 2^22 elements).
POPE_LIN_HD uint32_t lin_step(const LinRows& r) { return (uint32_t)r.s[2] * lin_size(r.type); }

// Rows of a call with n of them.  A single row's stride may be anything, and is nothing here: the jobs that go over the rows in
// reverse count from a row in front of the first, with a stride of 32 bits back to it.
inline LinRows lin_rows(const void* p, const int64_t* s, int n, int cols, int type, int unit) {
  LinRows r;
  r.p = const_cast<void*>(p);
  r.s[0] = s[0], r.s[1] = s[1], r.s[2] = n > 1 ? s[2] : 0;
  r.cols = cols;
  r.type = type;
  const int own = unit * lin_size(type), whole = own < 16 ? own : 16;   // bytes of an access
  r.vec = cols % unit == 0 && reinterpret_cast<uintptr_t>(p) % whole == 0 && r.s[0] % unit == 0 && r.s[1] % unit == 0 && r.s[2] % unit == 0;
  return r;
}

}  // namespace pope
