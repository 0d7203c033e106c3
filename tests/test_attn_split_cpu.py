"""How tg_attention_shared cuts its work (csrc/tg_attn_split.h), compiled for the
host with the sanitizer of undefined behaviour: no division by zero, no
conversion of a number that does not fit, for empty batches and any count of SMs."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "tinygiant_b200" / "csrc"
MAIN = """
#include "tg_attn_split.h"
#include <cstdio>
int main() {
  const int sizes[][3] = {{64, 8, 64}, {32, 4, 128}, {128, 1, 64}, {48, 2, 128}, {5, 5, 8}, {200, 200, 96}};
  long long n = 0;
  for (int sms : {1, 2, 7, 8, 15, 132, 148, 152, 160})
    for (int B : {0, 1, 3, 64, 1000})
      for (int P : {0, 1, 128, 129, 5000, 1 << 20})
        for (int len : {0, 1, 127, 4096, 1 << 20})
          for (auto& z : sizes) {
            const tg::SharedSplit s(B, P, len, z[0], z[1], z[2], sms);
            const long long blocks = (P + 127) / 128, stages = (long long)B * z[1] * s.ngc * ((len + 127) / 128);
            const bool pieces = B && P ? s.nsp >= 1 && s.nsp <= blocks : s.nsp == 0;
            const bool own = B && len ? s.own_ctas >= 1 && s.own_ctas <= sms && s.own_ctas <= stages : s.own_ctas == 0;
            if (!pieces || !own) {
              std::printf("batch %d prefix %d len %d heads %d/%d x %d sms %d: %d pieces, %d own\\n", B, P, len, z[0], z[1], z[2], sms, s.nsp,
                          s.own_ctas);
              return 1;
            }
            n++;
          }
  std::printf("%lld\\n", n);
}
"""


@pytest.mark.skipif(not shutil.which("g++"), reason="no g++")
def test_the_split_is_defined_for_every_size(tmp_path):
    (tmp_path / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined,float-cast-overflow,float-divide-by-zero",
                    "-fno-sanitize-recover=all", "-I", str(CSRC), str(tmp_path / "main.cpp"), "-o", str(tmp_path / "split")], check=True)
    r = subprocess.run([str(tmp_path / "split")], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert int(r.stdout) == 9 * 5 * 6 * 5 * 6


def test_the_workspace_of_an_empty_batch(lib):
    """A prefix and a cache, but no sequence: no workspace, and the call is one that does nothing."""
    for H, KH, hd in ((64, 8, 64), (32, 4, 128)):
        for weights in (0, 1):
            assert lib.tg_attention_shared_workspace(0, 16384, 1024, H, KH, hd, weights) == 0
    st = (ctypes.c_int64 * 16)(*[64] * 16)
    buf = (ctypes.c_float * 64)()
    p = ctypes.addressof(buf)
    assert lib.tg_attention_shared(0, p, p, p, p, p, p, p, None, None, 0, 16384, 1024, 1024, 32, 4, 64, st, 0, 0.125, None, 0, None) == 0
