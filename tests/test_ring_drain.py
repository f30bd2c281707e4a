"""The products' load warps leave no arrival behind that nobody has waited for: tcgen05.commit arrives on the stages'
barriers by itself, in the peer CTA's shared memory too, and a CTA's shared memory goes to the next one when it ends.
The kernels' own end-of-ring rule (csrc/ring.h) runs here against model barriers whose arrivals come as late as they
can: only when something waits for them."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "logic-bs-roformer-rs_b200" / "csrc"

MODEL = r"""
#include <cstdio>
#include <cstdlib>
#include <deque>
#include "ring.h"

// A ring of S stages: uses fill them in order, each use's arrival comes once something cannot go on without it.
template <int S>
struct Ring {
  unsigned done[S] = {};      // completed phases of each stage's barrier
  std::deque<int> pending;    // stages whose arrivals are under way, in order
  bool test(int s, unsigned parity) const { return (done[s] & 1u) != parity; }
  bool wait(int s, unsigned parity) {
    while (!test(s, parity)) {
      if (pending.empty()) return false;  // would wait for good
      ++done[pending.front()];
      pending.pop_front();
    }
    return true;
  }
};

template <int S>
void check(unsigned uses) {
  Ring<S> r;
  for (unsigned u = 0; u < uses; ++u) {
    if (!r.wait(u % S, ((u / S) & 1u) ^ 1u)) { printf("use %u of %u waits for good, %d stages\n", u, uses, S); exit(1); }
    r.pending.push_back(u % S);
  }
  if (r.pending.size() != (uses < S ? uses : S)) { printf("the model's arrivals are not late\n"); exit(1); }
  const bool ok = lbrr::drain_ring<S>(uses, [&](int s, uint32_t parity) { return r.wait(s, parity); });
  if (!ok || !r.pending.empty()) { printf("%zu arrivals left after %u uses of %d stages\n", r.pending.size(), uses, S); exit(1); }
  // a wait that gives up ends the drain
  unsigned calls = 0;
  if (uses > 1 && (lbrr::drain_ring<S>(uses, [&](int, uint32_t) { return ++calls < 2; }) || calls != 2)) exit(2);
}

int main() {
  for (unsigned uses = 0; uses < 200; ++uses) check<3>(uses), check<4>(uses);
  check<4>(1000003);
  check<3>(1000001);
  puts("ok");
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_no_arrival_is_left(tmp_path):
    (tmp_path / "model.cpp").write_text(MODEL)
    exe = tmp_path / "model"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(CSRC), str(tmp_path / "model.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


@pytest.mark.parametrize("source", ["gemm8.cu", "gemm8_few.cuh"])
def test_both_products_drain_their_ring(source):
    """In the load warp's branch, after its loop."""
    text = (CSRC / source).read_text()
    load = text[text.rindex("if (warp == ", 0, text.index("drain_ring<")):text.index("drain_ring<")]
    assert "LoadWarp" in load and "for (" in load
