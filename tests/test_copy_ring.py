"""The order of the copy ring's loads, waits and stores (csrc/copy_ring.cuh), run on the CPU with a wait that runs out at any place."""
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "nano_vllm_b200" / "csrc"

HARNESS = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "copy_ring.cuh"

constexpr int STAGES = 6, LEAD = 2;
// A stage's loads complete in order; the barrier's phase says how many have.  Wait number `late` runs out while its load is under
// way; a later wait for the same load finds it.
struct Io {
  int late, waits = 0, reads = 0;
  std::vector<int> in_flight = std::vector<int>(STAGES), loads = in_flight, full = in_flight;
  std::vector<int> storing;  // stages whose stores may still read, oldest first
  std::vector<int> out;      // pieces stored
  std::vector<int> holds = in_flight;
  void need(bool cond, const char* what) {
    if (!cond) { std::printf("%s\n", what); std::exit(1); }
  }
  template <int N>
  void read() {
    while (static_cast<int>(storing.size()) > N) storing.erase(storing.begin());
  }
  void load(int s, int piece) {
    for (int o : storing) need(o != s, "a load into a stage that a store still reads");
    need(!in_flight[s] && !full[s], "a load into a stage that holds a piece");
    in_flight[s] = 1;
    holds[s] = piece;
    ++loads[s];
  }
  bool wait(int s, uint32_t parity) {
    need(loads[s] > 0 && parity == static_cast<uint32_t>((loads[s] - 1) & 1), "a wait for another phase than the last load's");
    if (waits++ == late) return false;
    if (in_flight[s]) full[s] = 1;
    in_flight[s] = 0;
    return true;
  }
  void store(int s) {
    need(full[s], "a store of a piece that is not there");
    full[s] = 0;
    storing.push_back(s);
    out.push_back(holds[s]);
  }
  void finish() { storing.clear(); }
};

int main() {
  for (int pieces = 0; pieces < 40; ++pieces)
    for (int late = -1; late < pieces; ++late) {
      Io io{late};
      nvllm::CopyRing<STAGES, LEAD, Io> ring{io};
      for (int i = 0; i < pieces && ring.ok; ++i) ring.piece(i);
      const bool ok = ring.end();
      io.need(ok == (late < 0), "the wait that ran out is not told");
      for (int s = 0; s < STAGES; ++s) io.need(!io.in_flight[s], "a load is under way at the end");
      io.need(io.storing.empty(), "a store is under way at the end");
      io.need(static_cast<int>(io.out.size()) == (late < 0 ? pieces : late), "other pieces than those before it were stored");
      for (size_t i = 0; i < io.out.size(); ++i) io.need(io.out[i] == static_cast<int>(i), "pieces out of order");
    }
  return 0;
}
"""


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    folder = tmp_path_factory.mktemp("ring")
    source = folder / "ring.cpp"
    source.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", str(source), "-o", str(folder / "ring")], check=True)
    return folder / "ring"


def test_nothing_is_in_flight_when_a_ring_ends(harness):
    done = subprocess.run([str(harness)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout
