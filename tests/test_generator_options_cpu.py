"""CPU: the generator of the ViT attention body takes the options it has and no others."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

GEN = os.path.join(ROOT, "tools", "gen_attn_p2.py")


def generate(tmp_path, *opts):
    out = tmp_path / "body.inc"
    env = {**{k: v for k, v in os.environ.items() if not k.startswith("UFV_")}, "UFV_P2_OUT": str(out)}
    return subprocess.run([sys.executable, GEN, *opts], env=env, capture_output=True, text=True), out


@pytest.mark.parametrize("opts", [("--stamps",), ("--seq",), ("--seq", "x"), ("--seq=",), ("729",), ("--simple", "--seqq=729")])
def test_unknown_options_are_refused(tmp_path, opts):
    r, out = generate(tmp_path, *opts)
    assert r.returncode != 0 and "usage" in r.stderr and not out.exists()


@pytest.mark.parametrize("opts", [(), ("--simple",), ("--seq", "729"), ("--seq=729",), ("--seq=576", "--simple")])
def test_known_options_are_taken(tmp_path, opts):
    r, out = generate(tmp_path, *opts)
    assert r.returncode == 0 and out.read_text().startswith("// GENERATED by tools/gen_attn_p2.py")


def test_the_variant_builder_passes_no_other_options():
    text = open(os.path.join(ROOT, "tools", "lab", "build_p2_variants.sh")).read()
    assert "gen_attn_p2.py > /dev/null" in text and "--stamps" not in text and "_st" not in text
