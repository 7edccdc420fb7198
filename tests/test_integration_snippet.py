"""The C sequence that INTEGRATION.md shows for experts in 8-bit floating point: it compiles against the public header, every buffer
that a step reads is the caller's or written by an earlier step, and the slots are cleared before the down product."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# what the host owns: inputs, and room for each step's results, of the types that the operators write
HOST = """
#include <stddef.h>
#include "inzg.h"
int cudaMemsetAsync(void *, int, size_t, void *);
void inz_die(const char *, ...);
void layer(inzg_ctx *ctx, int l, int n, int H, int FF, int E, int K, void *st, const float *x, float *res, const float *norm,
           const void *gu8, const float *gus, const void *dn8, const float *dns, float *xn, void *xq, float *xs, int32_t *sel,
           float *w, int32_t *off, int32_t *rows, int32_t *slots, float *lw, void *h, void *hq, float *hs, float *slot_out, float *y) {
%s
}
"""


def _snippet():
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    return next(b for b in re.findall(r"```c\n(.*?)```", text, re.S) if "inzg_expert_lists" in b)


def test_the_sequence_compiles(tmp_path):
    gcc = shutil.which("gcc", path="/usr/bin") or shutil.which("gcc")
    if not gcc:
        pytest.skip("no C compiler")
    src = tmp_path / "layer.c"
    src.write_text(HOST % _snippet())
    r = subprocess.run([gcc, "-std=c11", "-Wall", "-Wextra", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(src)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_the_rows_that_are_routed_are_the_norms_fp32_result():
    text = _snippet()
    norm = re.search(r"inzg_rmsnorm_q8_args \w+ = \{(.*?)\};", text, re.S).group(1)
    assert ".type = INZG_T_F32" in norm and ".y = xn," in norm and re.search(r"inzg_route\(ctx, l, n, xn,", text)


def test_the_slots_are_cleared_before_the_down_product():
    text = _snippet()
    clear, down = text.index("cudaMemsetAsync(slot_out, 0,"), text.index("inzg_grouped_matmul(ctx, &dn)")
    assert clear < down < text.index("inzg_combine(")
