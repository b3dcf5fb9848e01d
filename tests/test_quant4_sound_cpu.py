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
