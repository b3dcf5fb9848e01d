"""Weights in 4 bits where no GPU is needed: what a wait that ran out is called, which bytes a step reads, what the command line says."""
from __future__ import annotations

import re

import pytest

import moe_b200.ops.build as build


def test_a_wait_is_called_by_its_own_name():
    """Every site that the kernels of few rows report has a role of that kernel's, no tensor-core role of the same number."""
    from moe_b200.ops import core

    with open(f"{build.CSRC}/gemm_q4.cu", encoding="utf-8") as f:
        sites = sorted({int(s, 16) for s in re.findall(r"0x6[0-9a-f](?![0-9a-f])", f.read())})
    assert sites == [0x61, 0x62, 0x63, 0x64]
    for site, word in zip(sites, ("free stage", "in flight", "picks", "loaded stage")):
        text = core.wait_site(site)
        assert word in text and "MMA" not in text and "few rows" in text, text
    assert "MMA issuer" in core.wait_site(0x53)


@pytest.mark.parametrize("options", [["--weights", "int3"], ["--weights", "int4", "--weight-group", "48"]])
def test_info_refuses_weights_that_there_are_none_of(model_dirs, options, capsys):
    from moe_b200 import cli

    d = model_dirs.get("A", "bfloat16", seed=1, std=0.02)
    with pytest.raises(SystemExit):
        cli.main(["info", d, *options])
    assert "weight" in capsys.readouterr().err
    assert cli.main(["info", d, "--weights", "int4"]) == 0


def test_a_copy_of_a_weight_is_a_weight_of_its_own_tensors():
    """Copied, and stored and read back: the addresses that kernels are given are those of the copy's tensors, and nobody has read them yet."""
    import copy
    import pickle

    import test_quant4_cpu as T

    w = T._w((3, 32, 70), 32, pair=True)
    w.settle()
    for c in (copy.deepcopy(w), pickle.loads(pickle.dumps(w))):
        assert c.pointers == (c.codes.data_ptr(), c.scales.data_ptr()) and c.codes.data_ptr() != w.codes.data_ptr()
        assert (c.shape, c.group, c.pair, c.place) == (w.shape, w.group, w.pair, w.place) and c.read_on == ()
        assert bool((c.codes == w.codes).all())
    assert copy.copy(w).codes is w.codes
