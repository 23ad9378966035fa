"""The host arithmetic of the pair-stream kernels, compiled from their header and run on the CPU: quotients by multiplication, the form
of a tensor with axes of one entry, grids."""
import random
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "fold_cp_ops_b200" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include "pair_stream.cuh"
using namespace pair;
int main() {
  char what;
  while (scanf(" %c", &what) == 1) {
    if (what == 'q') {
      unsigned n, d;
      if (scanf("%u %u", &n, &d) != 2) return 1;
      printf("%u\n", make_fast_div(d).div(n));
    } else if (what == 'c') {
      pair_tensor_t t = {&what, 0, 0, 0};
      int b, i, j;
      long long sb, si, sj;
      if (scanf("%d %d %d %lld %lld %lld", &b, &i, &j, &sb, &si, &sj) != 6) return 1;
      t.stride_b = sb, t.stride_i = si, t.stride_j = sj;
      const pair_tensor_t c = canonical(&t, b, i, j);
      printf("%lld %lld %lld %d\n", (long long)c.stride_b, (long long)c.stride_i, (long long)c.stride_j, (int)collapses(&c, i, j));
    } else if (what == 'g') {
      unsigned long long need;
      int sms, resident;
      unsigned steps;
      if (scanf("%llu %d %d %u", &need, &sms, &resident, &steps) != 4) return 1;
      printf("%u\n", walk_grid(need, sms, resident, steps));
    }
  }
  const pair_tensor_t none = canonical(nullptr, 1, 1, 1);
  return none.data == nullptr && collapses(&none, 1, 1) ? 0 : 2;
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(nvcc).exists():
        pytest.skip("no nvcc")
    at = tmp_path_factory.mktemp("host_arithmetic")
    (at / "main.cu").write_text(PROGRAM)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-diag-suppress", "177", "-I", str(CSRC), str(at / "main.cu"),
                    "-o", str(at / "main")], check=True, capture_output=True)

    def run(lines):
        done = subprocess.run([str(at / "main")], input="\n".join(lines), check=True, capture_output=True, text=True)
        return [tuple(int(v) for v in line.split()) for line in done.stdout.splitlines()]

    return run


def test_quotients_by_multiplication(ask):
    rng, asked = random.Random(2), []
    divisors = [1, 2, 3, 5, 7, 8, 96, 197, 1023, 1024, 1025, 65535, 65536, (1 << 30) - 1, 1 << 30, (1 << 30) + 1, (1 << 31) - 1]
    for d in divisors + [rng.randrange(1, 1 << 31) for _ in range(500)]:
        ns = [0, 1, d - 1, d, (1 << 31) - 1] + [rng.randrange(1 << 31) for _ in range(20)]
        ns += [k for q in (1, 5, ((1 << 31) - 1) // d) for k in (q * d - 1, q * d) if 0 <= k < 1 << 31]
        asked += [(n, d) for n in ns]
    assert ask([f"q {n} {d}" for n, d in asked]) == [(n // d,) for n, d in asked]


def test_axes_of_one_entry_have_the_stride_that_lets_rows_follow_one_another(ask):
    rng, asked, odd = random.Random(3), [], 12345677
    for _ in range(2000):
        shape = [rng.choice((1, 1, 2, 3, 7)) for _ in range(3)]
        strides, step = [], rng.choice((8, 64, 128))
        for n in reversed(shape):
            strides.insert(0, step if n > 1 else odd)
            step *= n
        if rng.random() < 0.5:  # a gap somewhere
            axis = rng.randrange(3)
            strides[axis] += 8
        asked.append((shape, strides))
    for (shape, strides), (sb, si, sj, flat) in zip(asked, ask(["c " + " ".join(map(str, s + t)) for s, t in asked])):
        rows = [(b, i, j) for b in range(shape[0]) for i in range(shape[1]) for j in range(shape[2])]
        at = [sum(k * s for k, s in zip(row, strides)) for row in rows]
        assert at == [b * sb + i * si + j * sj for b, i, j in rows]
        distance = at[1] if len(at) > 1 else 0
        assert flat == (at == [k * distance for k in range(len(at))]), (shape, strides)
        assert all(s % 8 == 0 for s in (sb, si, sj)), "an axis of one entry says nothing about alignment"


def test_grids_are_one_wave_or_whole_waves_of_about_so_many_steps(ask):
    """A grid is rounded to the nearest wave: at most half a wave more CTAs than need / steps."""
    rng = random.Random(4)
    asked = [(rng.choice((1, 147, 148, 1184, 1185, rng.randrange(1, 1 << 20), rng.randrange(1, 1 << 31))), 148, rng.randrange(1, 17), rng.choice((1, 4, 8, 32)))
             for _ in range(2000)]
    for (need, sms, resident, steps), (grid,) in zip(asked, ask(["g " + " ".join(map(str, a)) for a in asked])):
        wave = sms * resident
        if need <= wave:
            assert grid == need
        else:
            assert grid % wave == 0 and (grid == wave or abs(grid - need // steps) <= wave / 2)
