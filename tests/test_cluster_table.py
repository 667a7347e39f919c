"""The table of how many clusters of a kernel fit (csrc/cluster_table.h) on
the host, with a fake of the question that it asks the device."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <initializer_list>
#include "cluster_table.h"

static int asked = 0;
static int fit(s3::ClusterTable& t, int dev, int n, int answer, int status) {
  return t.fit(dev, n, [&](int* f) { ++asked; *f = answer; return status; });
}
#define WANT(x) if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; }

int main() {
  static s3::ClusterTable t, other;
  WANT(fit(t, 0, 8, 15, 0) == 15 && asked == 1);
  WANT(fit(t, 0, 8, 99, 0) == 15 && asked == 1);   // kept
  WANT(fit(t, 1, 8, 7, 0) == 7 && asked == 2);     // another device is asked for itself
  WANT(fit(t, 0, 8, 99, 0) == 15 && asked == 2);
  WANT(fit(t, 0, 16, 4, 0) == 4 && asked == 3);    // and so is another size
  WANT(fit(other, 0, 8, 3, 0) == 3 && asked == 4); // and another kernel
  WANT(fit(t, 2, 8, 5, 1) == 0 && asked == 5);     // a failed question: nothing fits,
  WANT(fit(t, 2, 8, 5, 0) == 5 && asked == 6);     //   once
  WANT(fit(t, 3, 8, 0, 0) == 0 && asked == 7);     // none is an answer
  WANT(fit(t, 3, 8, 9, 0) == 0 && asked == 7);
  for (int dev : {-1, 64, 1000}) {                 // not in the table: asked each time
    const int before = asked;
    WANT(fit(t, dev, 2, 6, 0) == 6 && fit(t, dev, 2, 6, 0) == 6 && asked == before + 2);
  }
  WANT(fit(t, 63, 16, 2, 0) == 2 && fit(t, 63, 16, 0, 0) == 2);
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler")
def test_cluster_table(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "sam3.c_b200", "csrc"), str(src),
                    "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
