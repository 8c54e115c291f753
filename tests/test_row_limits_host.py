"""Row arithmetic of the attention kernels near 2^31 (tempo_amd/csrc/row_limits.h), compiled for the host and compared
with the same in 64 bits."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

# the most rows a table may have, and smaller ones; every function sees each pair of rows that its kernel forms
PROGRAM = r"""
#include <stdio.h>
#include <stdlib.h>
#include <vector>
#include "row_limits.h"
using namespace tmp;
typedef long long ll;
static long checked = 0;
static void expect(ll got, ll want, const char *what, ll a, ll b, ll c) {
  ++checked;
  if (got != want) { printf("%s(%lld, %lld, %lld) = %lld, expected %lld\n", what, a, b, c, got, want); exit(1); }
}
int main() {
  const ll most = (1ll << 31) - 65537;
  for (ll n : {1ll, 130ll, 5000ll, 1ll << 30, (1ll << 30) + 77, 1200000000ll, most - 64, most}) {
    std::vector<ll> rows, sizes;
    for (ll base : {0ll, n / 7, n / 2, n - n / 9, n})
      for (ll d : {-129ll, -128ll, -64ll, -1ll, 0ll, 1ll, 63ll, 64ll, 127ll})
        if (base + d >= 0 && base + d < n + 128) rows.push_back(base + d);
    for (ll s : {1ll, 2ll, 64ll, 1000ll, n / 3, n / 2, n - 1, n})
      if (s >= 1 && s <= n) sizes.push_back(s);
    BODY
  }
  printf("%ld comparisons\n", checked);
}
"""

BODIES = {
    # query rows r of key rows j: of the key's tile or behind it
    "window": r"""
    for (ll j : rows) for (ll w : sizes) {
      if (j < n) expect(window_end((int)j, 128, (int)w, (int)n), j + 128 + w - 1 < n ? j + 128 + w - 1 : n, "window_end", j, w, n);
      for (ll r : rows) {
        if (r < j - 128) continue;
        expect(beyond_window((int)r, (int)j, (int)w), r > j + w - 1, "beyond_window", r, j, w);
        expect(window_reach((int)j, (int)r, (int)w), j + w - 1 - r, "window_reach", j, r, w);
      }
    }""",
    "section": r"""
    for (ll s : sizes) for (ll first : rows) {
      if (first >= n) continue;
      expect(section_end((int)first, (int)s, (int)n), first + s < n ? first + s : n, "section_end", first, s, n);
    }""",
}


@pytest.mark.parametrize("what", list(BODIES))
def test_rows_near_the_largest_table(what, tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc to compile the header with")
    src, exe = tmp_path / "rows.hip", tmp_path / "rows"
    src.write_text(PROGRAM.replace("BODY", BODIES[what]))
    # (signed overflow is made an error of the run, so that a sum which happens to wrap back shows as well)
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O1", "-Xarch_host", "-fsanitize=signed-integer-overflow", "-Xarch_host",
                    "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "tempo_amd", "csrc"), str(src), "-o", str(exe)],
                   check=True, capture_output=True, timeout=300)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout + run.stderr
    assert int(run.stdout.split()[0]) > 500
