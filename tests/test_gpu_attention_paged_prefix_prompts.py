"""Prompts of hundreds and thousands of tokens behind a shared prefix, alone and beside single tokens, against the definition in 64 bits: rows of many joining CTAs, tokens of many blocks."""
import pytest

torch = pytest.importorskip("torch")
from test_gpu_attention_paged_prefix import TYPES, one  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,held", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (7, 1)])
def test_a_prompt_of_hundreds(dev, pkg, dtype, held, d, hq, hkv):
    one(pkg, dev, 41, [(700, 700)], hq, hkv, d, 16, dtype, held, 20)


@pytest.mark.parametrize("held", ["bf16", "i8"])
def test_a_prompt_of_thousands(dev, pkg, held):
    one(pkg, dev, 42, [(2500, 2611)], 32, 8, 128, 64, "bf16", held, 5)


@pytest.mark.parametrize("dtype,held", TYPES)
def test_prompts_beside_single_tokens(dev, pkg, dtype, held):
    one(pkg, dev, 43, [(1, 90), (900, 1300), (0, 5), (1, 1), (300, 300), (64, 64), (5, 700)], 16, 4, 128, 32, dtype, held, 70, gap=3)


@pytest.mark.parametrize("held", ["bf16", "i8"])
def test_rows_whose_records_are_many(dev, pkg, held):
    """Few heads and rows on a long prefix: sixteen groups of threads join a row."""
    one(pkg, dev, 44, [(3, 40)], 2, 1, 128, 64, "bf16", held, 400)
    one(pkg, dev, 45, [(12, 40), (1, 9)], 2, 1, 64, 64, "bf16", held, 400)
