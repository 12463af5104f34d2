"""Attention over a paged cache where it is easily wrong: work without keys, values at the ends of the types, rarely taken paths."""
import pytest

from conftest import pulpnn

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from test_gpu_attention import BF16, F16, _settled, prompt_case  # noqa: E402, F401

api = pulpnn.api


# ---- prompts: queries that see no key, more of them than the GPU takes at once ------------------------------

@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("with_keys", ["first", "last", "every third", "none"])
def test_prompt_many_sequences_without_keys(dtype, dim, with_keys):
    """600 sequences of one query, in the sequences' order: a CTA meets several in a row that have no keys."""
    has = {"first": lambda b: b < 148, "last": lambda b: b >= 452, "every third": lambda b: b % 3 == 1, "none": lambda b: False}[with_keys]
    prompt_case(21, [1] * 600, [(b * 7) % 200 if has(b) else -1 for b in range(600)], 1, 1, dim, dtype)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("few", [0, 1, 3])
def test_prompt_sequences_without_keys_longest_first(dtype, dim, few):
    """256 sequences of several lengths, taken longest first: those without keys lie among the others."""
    lens = [1 + (b * 37) % 300 if b % 4 == few else 1 + b % 3 for b in range(256)]
    prompt_case(22, lens, [-n if (b // 4) % 2 else 0 for b, n in enumerate(lens)], 8, 8, dim, dtype)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
def test_prompt_with_fewer_keys_than_queries(dtype, dim):
    """4096 queries on 2000 keys: the first half sees none. Then 20 sequences, longest first."""
    prompt_case(23, [4096], [2000 - 4096], 32, 8, dim, dtype)
    prompt_case(24, [700] * 20, [-600] * 20, 32, 8, dim, dtype)


def test_prompt_all_at_once_and_without_keys():
    """No more units than SMs, each an item of its own."""
    prompt_case(25, [1, 140] * 20, [-1, -140, 3, 0] * 10, 2, 2, 64, BF16)
