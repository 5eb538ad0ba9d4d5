// Host check of the slot and scale arithmetic of the 8-bit pages (no GPU code runs).
#include <math.h>
#include <stdio.h>

#include "../quashkv_b200/csrc/paged8.cuh"

using namespace qkv::p8;

template <int CODE> static int check_scales(float most) {
  int bad = 0;
  for (int e = -149; e < 128; ++e)
    for (float m : {1.f, 1.0000001f, 1.5f, 1.75f, 1.7500001f, 1.984375f, 1.9843751f, 1.9999999f}) {
      const float top = ldexpf(m, e), s = scale_for<CODE>(top);
      if (top == 0.f) continue;
      int k;
      if (frexpf(s, &k) != 0.5f) ++bad;                                   // a power of two
      if (!(top <= most * static_cast<double>(s))) ++bad;                 // that holds the largest
      if (k - 1 > kLeastExp && top <= most * static_cast<double>(s) / 2) ++bad;      // and is the least one
      if (k - 1 < kLeastExp) ++bad;
    }
  if (scale_for<CODE>(0.f) != 0.f) ++bad;
  if (!isnan(scale_for<CODE>(INFINITY)) || !isnan(scale_for<CODE>(NAN))) ++bad;
  return bad;
}

int main() {
  int bad = check_scales<kE4M3>(448.f) + check_scales<kInt8>(127.f);
  const int32_t row[4] = {7, -1, 2147483647, 0};
  for (int bs : {16, 48, 128})
    for (int64_t pos = -2; pos < 5 * bs; ++pos) {
      const int64_t s = slot_of(row, 4, bs, pos);
      const int64_t want = pos < 0 || pos >= 4 * bs || row[pos / bs] < 0 ? -1 : static_cast<int64_t>(row[pos / bs]) * bs + pos % bs;
      if (s != want) ++bad;
    }
  if (bad) { printf("%d wrong\n", bad); return 1; }
  printf("paged8 host checks OK\n");
  return 0;
}
