// Addresses of rows as the linear attention's kernels form them (csrc/linear_rows.hpp: a base in 64 bits, an offset from it in 32), walked on
// the host over both directions, chunks, lengths and strides: every access is to a row of the segment, also where a call's only
// row has a stride that would be far outside.
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "linear_rows.hpp"

using namespace pope;

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); std::exit(1); } } while (0)

int main() {
  alignas(16) static char memory[16];
  const int64_t most = ((int64_t)1 << 22) - 1;
  for (const int type : {0, 1, 2})
    for (const int N : {1, 2, 31, 32, 33, 63, 64, 65, 129, 200, 700})
      for (const int64_t stride : {(int64_t)0, (int64_t)64, (int64_t)65, most, (int64_t)1 << 25, ((int64_t)1 << 26) + 8, (int64_t)1 << 31, ((int64_t)1 << 40) + 1}) {
        if (N > 1 && stride > most) continue;   // refused
        const int64_t s[3] = {64, 64, stride};
        const LinRows r = lin_rows(memory, s, N, 64, type, 8);
        CHECK(r.s[2] == (N > 1 ? stride : 0));
        CHECK(r.vec == (N == 1 || stride % 8 == 0));
        const uint32_t step = lin_step(r);
        const int64_t size = lin_size(type);
        for (const int L : {64, 192})
          for (int row0 = 0; row0 < N; row0 += L) {
            const int len = N - row0 < L ? N - row0 : L;
            for (const int C : {32, 64})
              for (const bool rev : {false, true})
                for (int t0 = 0; t0 < len; t0 += C) {
                  const int64_t base = ((int64_t)row0 + (rev ? len - C - t0 : t0)) * r.s[2] * size;
                  for (int t = 0; t < C; ++t) {
                    const int at = t < len - 1 - t0 ? t : len - 1 - t0;   // rows behind the segment are the last one's again
                    const uint32_t place = rev ? C - 1 - at : at;
                    const int64_t row = rev ? row0 + len - 1 - t0 - at : row0 + t0 + at;
                    CHECK(row >= row0 && row < row0 + len);
                    CHECK(base + (int64_t)(uint32_t)(place * step) == row * r.s[2] * size);
                  }
                }
            for (int r0 = 0; r0 < len; r0 += 256)   // the queries' expansion
              for (int t = 0; t < 256; ++t) {
                const int at = t < len - r0 - 1 ? t : len - r0 - 1;
                CHECK(((int64_t)row0 + r0) * r.s[2] * size + (int64_t)(uint32_t)(at * step) == ((int64_t)row0 + r0 + at) * r.s[2] * size);
              }
          }
      }
  std::printf("ok\n");
}
