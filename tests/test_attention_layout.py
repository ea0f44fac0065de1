"""What the host says of an attention plan's list before any lengths are known, by a program of its own over the library's headers."""
import os
import shutil
import subprocess

import pytest

from valora_amd import _build

PROGRAM = """
#include <cstdio>
#include <cstdlib>
#include "attention.h"
int main(int n, char **v) {
  for (int i = 1; i + 2 < n; i += 3) {
    mlora_attention_plan p{};
    p.n_req = atoi(v[i]);
    p.n_tokens = atoi(v[i + 1]);
    p.kv_heads = p.q_heads = atoi(v[i + 2]);
    p.max_seq_len = 1;
    p.max_kv_len = 70000;
    p.head_dim = 128;
    p.page_size = 2;
    printf("%d", (int)mlora::attention_layout(p).few_whole);
  }
}
"""


def test_requests_are_whole_by_those_that_have_new_tokens(tmp_path):
    """A cache's slots without new tokens do not make a pass's few requests many."""
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    (tmp_path / "p.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__=1", "-I/opt/rocm/include", "-I", os.path.join(_build.ROOT, "include"), "-I", _build.CSRC,
                    str(tmp_path / "p.cpp"), _build.LIB_PATH, "-L/opt/rocm/lib", "-lamdhip64", f"-Wl,-rpath,{_build.HERE}:/opt/rocm/lib",
                    "-o", str(tmp_path / "p")], check=True)
    cases = [(256, 5, 8, 0), (256, 127, 8, 0), (256, 128, 8, 1), (128, 128, 8, 1), (127, 4000, 8, 0), (5, 5, 8, 0), (1024, 1024, 1, 1), (1 << 20, 32, 32, 1),
             (1 << 20, 31, 32, 0)]
    out = subprocess.run([str(tmp_path / "p")] + [str(x) for c in cases for x in c[:3]], check=True, capture_output=True, text=True).stdout
    assert out == "".join(str(c[3]) for c in cases)
