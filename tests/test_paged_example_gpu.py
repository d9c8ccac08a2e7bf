"""The generation example: append, attention and read together over many steps."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_generation.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_generation", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("flags", [
    [],
    ["--window", "0", "--page", "32", "--group", "1", "--group-mode", "bands4"],
    ["--window", "100", "--sink", "20", "--k-bits", "8", "--v-bits", "8", "--page", "64", "--common", "130"],
    ["--window", "33", "--sink", "0", "--k-bits", "8", "--group-mode", "bands", "--step-tokens", "60", "--batch", "5"],
])
def test_every_attention_agrees_with_a_dense_one(example, flags):
    """Relative error of each layer's and step's output in the 2-norm: output rounding to bf16
    (at most 2^-8 of an element, about 2^-9.8 rms), weights and int8 products to fp16."""
    a = example.parse(["--check", "--layers", "2", "--heads", "2", "--requests", "9", "--prompt", "300", "--out", "12",
                       "--pages", "600", *flags])
    r = example.generate(a)
    assert r["requests"] == 9 and all(len(o) >= 1 for o in r["outputs"])
    assert 0 < r["worst"] < 2.0 ** -8


def test_same_tokens_again(example):
    """The same requests in the same steps give the same tokens: no result depends on the
    order in which blocks ran."""
    a = example.parse(["--layers", "2", "--heads", "2", "--requests", "6", "--prompt", "400", "--out", "20", "--pages", "600"])
    assert example.generate(a)["outputs"] == example.generate(a)["outputs"]
