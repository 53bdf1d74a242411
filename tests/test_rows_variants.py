"""The launch shapes of the row operators' kernels that the compile check covers, without a GPU."""
import re

import pytest

import accelerate_b200 as A
from accelerate_b200 import backend


def variants(term, monkeypatch):
    """The defines of every variant of a one-node program, as the compile check lists them."""
    text, out = A.build_program(list(term)).text, []
    while True:
        monkeypatch.setenv("ACCELERATE_B200_SOURCE_VARIANT", str(len(out)))
        try:
            source = backend.kernel_source(text, 0)
        except backend.B200Error:
            return out
        out.append({m[1]: int(m[2]) for m in re.finditer(r"#define ((?:ROW|NORM)_\w+) (\d+)\n", source)})


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_every_number_of_ctas_per_row_is_compiled(lib_built, monkeypatch, t):
    """1 to 8 CTAs share a row of statistics and 1 to 16 one of the gradient, by the numbers of rows and SMs."""
    P = A.param
    x, ids, te = P(2, t), P(2, "i32"), P(2, "f32")
    for term, want in [(A.logProbs(5, P(1, "i32"), x), {1, 2, 4, 8}), (A.distill(2.0, ids, te, x), {1, 2, 4, 8}),
                       ([A.distillGrad(2.0, ids, te, x, P(1, "f32"), P(1, "f32"))], {1, 2, 4, 8, 16})]:
        got = [v["ROW_C"] for v in variants(term, monkeypatch)]
        assert set(got) == want and len(got) == len(want)


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_norms_are_compiled_for_few_rows_and_for_many(lib_built, monkeypatch, t):
    """A row of 1024 elements takes one or two warps where there are many rows, and up to eight where there are few."""
    P = A.param
    for term in (A.layerNorm(1e-5, P(1, "f32"), P(1, "f32"), P(2, t)), A.layerNormGrad(P(1, "f32"), P(2, t), P(1, ("f32", "f32")), P(2, t))):
        got = variants(term, monkeypatch)
        whole = [v for v in got if not v["NORM_LONG"] and not v.get("NORM_SUMS") and not v.get("NORM_COLS")]
        widest = max(v["NORM_VE"] for v in whole)
        shapes = {(v["NORM_WARPS"], v["NORM_U"]) for v in whole if v["NORM_VE"] == widest}
        assert any(u == 1 and warps > 1 for warps, u in shapes), "few rows: as many lanes as a row fills"
        assert any(u > 1 and warps <= 2 for warps, u in shapes), "many rows"
        assert len({tuple(sorted(v.items())) for v in got}) == len(got), "no variant twice"
