"""The 8-bit cache's codes, compiled for the host from the kernels' own header, against integers."""

import shutil
import subprocess

import pytest

from shrike_b200.ops import build

PROGRAM = """
#include "codes_q8.cuh"
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

// 127 x / a to the nearest integer, halves to even, for |x| <= a.
static int exact(float x, float a) {
  if (x == 0.f) return 0;
  int ex, ea;
  const __int128 X = static_cast<__int128>(ldexp(frexp(fabs(x), &ex), 24)), A = static_cast<__int128>(ldexp(frexp(a, &ea), 24));
  if (ea - ex > 60) return 0;
  const __int128 den = A << (ea - ex), num = 127 * X, whole = num / den, left = 2 * (num - whole * den);
  const int code = static_cast<int>(whole) + (left > den || (left == den && (whole & 1)) ? 1 : 0);
  return x < 0.f ? -code : code;
}

static uint64_t state = 88172645463325252ull;
static uint32_t random32() {
  state ^= state << 13; state ^= state >> 7; state ^= state << 17;
  return static_cast<uint32_t>(state >> 16);
}

int main() {
  long wrong = 0;
  auto look = [&](float x, float a) {
    if (fabsf(x) > a) return;
    for (const float y : {x, -x}) {
      const int got = cacheq8::code_of(y, a, 127.f / a);
      if (got != exact(y, a) && wrong++ < 5) printf("%a of %a: %d, not %d\\n", y, a, got, exact(y, a));
    }
  };
  look(0x1.1a3ba6p-8f, 0x1.18072ep+0f);
  const float special[] = {1.f, 2.f, 0x1.fffffep0f, 0x1.fcp0f, 1.5f, 0x1.000002p0f, 0x1.fc0002p0f, 0x1.fbfffep0f};
  for (int i = 0; i < 20000; ++i) {
    float a = i < 8 ? special[i] : 1.f + (random32() >> 9) * 0x1p-23f;
    const int shift[] = {0, -99, -20, 3, 40, 99};
    a = ldexpf(a, i < 48 ? shift[i / 8] : shift[random32() % 6]);
    for (int k = 0; k < 127; ++k) {   // every border, and two steps to either side of it
      float x = static_cast<float>(static_cast<double>(a) * (2 * k + 1) / 254);
      x = nextafterf(nextafterf(x, 0.f), 0.f);
      for (int step = 0; step < 5; ++step, x = nextafterf(x, INFINITY)) look(x, a);
    }
    for (int n = 0; n < 64; ++n) look(a * (random32() >> 8) * 0x1p-24f, a);
    look(a, a);
    look(0.f, a);
    look(nextafterf(a, 0.f), a);
    look(0x1p-126f, a);
  }
  if (wrong) printf("%ld wrong\\n", wrong);
  return wrong != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
def test_codes_of_32_bit_elements_fall_on_the_right_side_of_every_border(tmp_path):
    source, program = tmp_path / "codes.cpp", tmp_path / "codes"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-ffp-contract=off", "-x", "c++", f"-I{build.CSRC}", str(source), "-o", str(program)], check=True)
    run = subprocess.run([str(program)], stdout=subprocess.PIPE, text=True)
    assert run.returncode == 0, run.stdout
