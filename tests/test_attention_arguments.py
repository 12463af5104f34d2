"""Arguments of the attention entry points that the C structs cannot take: errors of the library, whatever the value."""
import pytest

from conftest import pulpnn
from test_attention_refusals import BF16, INVALID, S32, S8, UNSUPPORTED, cache, refused, rows

torch = pytest.importorskip("torch")
api = pulpnn.api
U8 = torch.uint8


def prompt(q=None, k=None, v=None, cu=None, out=None, **more):
    q = rows(7, 4, 64) if q is None else q
    k = rows(7, 2, 64) if k is None else k
    v = rows(7, 2, 64) if v is None else v
    cu = torch.tensor([0, 7], dtype=S32) if cu is None else cu
    api.pulpnn_attn_prompt(q, k, v, cu, rows(7, 4, 64) if out is None else out, **more)


def decode(q=None, table=None, lens=None, out=None, **more):
    api.pulpnn_attn_decode(cache(), rows(3, 4, 64) if q is None else q, torch.zeros(3, 2, dtype=S32) if table is None else table,
                           torch.zeros(3, dtype=S32) if lens is None else lens, rows(3, 4, 64) if out is None else out, **more)


@pytest.mark.parametrize("bad", [rows(7, 4, 64)[0], rows(7, 4, 64)[None], torch.zeros((), dtype=BF16)])
def test_rows_of_another_rank(bad):
    refused(INVALID, prompt, q=bad)
    refused(INVALID, prompt, k=bad)
    refused(INVALID, prompt, v=bad)
    refused(INVALID, prompt, out=bad)
    refused(INVALID, decode, q=bad)
    refused(INVALID, decode, out=bad)
    n, k = torch.arange(7), rows(7, 2, 64)
    refused(INVALID, api.pulpnn_kv_append, cache(), n, bad, k)
    refused(INVALID, api.pulpnn_kv_append, cache(), n, k, bad)
    refused(INVALID, api.pulpnn_kv_append, cache(), n, k, k, q=bad, q_out=rows(7, 4, 64))
    refused(INVALID, api.pulpnn_kv_append, cache(), n, k, k, q=rows(7, 4, 64), q_out=bad)
    refused(INVALID, api.pulpnn_kv_append, cache(), n, k, k, k_out=bad)
    refused(INVALID, api.pulpnn_kv_gather, cache(), n, bad)
    refused(INVALID, api.pulpnn_kv_gather, cache(), n, None, bad)


def test_vectors_of_another_rank():
    k, n = rows(6, 2, 64), torch.arange(6)
    one, many = torch.tensor(0), torch.zeros(2, 3, dtype=torch.int64)
    refused(INVALID, api.pulpnn_kv_append, cache(), one, k, k)
    for slots in (one, many):
        refused(INVALID, api.pulpnn_kv_gather, cache(), slots, k)
    for cu in (one.to(S32), many.to(S32)):
        refused(INVALID, prompt, cu=cu)
    refused(INVALID, prompt, cu=torch.zeros(0, dtype=S32))
    for freq in (torch.tensor(1.0, dtype=torch.float64), torch.ones(4, 8, dtype=torch.float64)):
        refused(INVALID, api.pulpnn_kv_append, cache(), n, k, k, positions=n.to(S32), inv_freq=freq)
    refused(INVALID, prompt, lse=torch.zeros(7, 4)[:, :, None])
    refused(INVALID, api.KVCache, torch.zeros(4, 16, 64, dtype=BF16), torch.zeros(4, 16, 64, dtype=BF16))
    codes = torch.zeros(4, 16, 2, 64, dtype=S8)
    refused(INVALID, api.KVCache, codes, codes, torch.zeros(4, 16), torch.zeros(4, 16))


def test_numbers_beyond_the_structs():
    for call in (prompt, decode):
        for window in (2 ** 31, -2 ** 31 - 1, 2 ** 70, 1.5, "3"):
            refused(INVALID, call, window=window)
        for scale in (1e39, -1e300, "1", 1j):
            refused(INVALID, call, scale=scale)
    q = rows(7, 4, 64)
    refused(INVALID, prompt, out=q.to(U8), out_step=1e39)
    refused(INVALID, prompt, out=q.to(U8), out_step=0.1, out_zero=2 ** 40)
    refused(INVALID, decode, out=q[:3].to(U8), out_step=0.1, out_zero=1.5)


def test_sizes_beyond_the_structs():
    n = 2 ** 31
    far = torch.zeros(1, 2, 64, dtype=BF16).expand(n, 2, 64)
    slots = torch.zeros(1, dtype=torch.int64).expand(n)
    refused(INVALID, api.pulpnn_kv_append, cache(), slots, far, far)
    refused(INVALID, prompt, k=far, v=far, cu_k=torch.tensor([0, 7], dtype=S32))


def test_prompts_of_too_many_sequences():
    refused(UNSUPPORTED, prompt, cu=torch.zeros(2 ** 24 + 2, dtype=S32), q=rows(7, 1, 64), k=rows(7, 1, 64), v=rows(7, 1, 64), out=rows(7, 1, 64))
    q, k = rows(7, 64, 64), rows(7, 8, 64)
    refused(UNSUPPORTED, prompt, cu=torch.zeros(2 ** 20 + 2, dtype=S32), q=q, k=k, v=k, out=q)
