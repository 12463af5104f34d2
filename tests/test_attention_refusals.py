"""What the attention entry points refuse, before they touch a GPU: every check of an argument comes ahead of the device's."""
import ctypes as C

import pytest

from conftest import pulpnn, _has_gpu

torch = pytest.importorskip("torch")
api = pulpnn.api
BF16, F16, F32, S32, S8 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.int8


def cache(dtype=BF16, pages=4, page=16, heads=2, dim=64, **more):
    k = torch.zeros(pages, page, heads, dim, dtype=dtype)
    if dtype == S8:
        s = torch.zeros(pages, page, heads)
        more = dict(k_scale=s, v_scale=s.clone(), **more)
    return api.KVCache(k, k.clone(), **more)


def refused(code, f, *a, **k):
    with pytest.raises(pulpnn.PulpNNError) as e:
        f(*a, **k)
    assert e.value.code == code, str(e.value)
    assert pulpnn.load_library().pulpnn_last_error() == 0


INVALID, UNSUPPORTED = api.ERR_INVALID_ARG, api.ERR_UNSUPPORTED


def rows(n, heads, dim, dtype=BF16):
    return torch.zeros(n, heads, dim, dtype=dtype)


def test_caches():
    k = torch.zeros(4, 16, 2, 64, dtype=BF16)
    refused(INVALID, api.KVCache, k, k[:3])
    refused(INVALID, api.KVCache, k, k.to(F16))
    refused(INVALID, api.KVCache, k, k.transpose(1, 2).contiguous().transpose(1, 2))
    refused(INVALID, api.KVCache, k.expand(4, 16, 2, 64).transpose(2, 3), k.transpose(2, 3))
    refused(INVALID, api.KVCache, k[:1].expand(4, 16, 2, 64), k[:1].expand(4, 16, 2, 64))
    refused(INVALID, api.KVCache, k.to(S8), k.to(S8))
    refused(INVALID, api.KVCache, k, k, torch.zeros(4, 16, 2), torch.zeros(4, 16, 2))
    refused(INVALID, api.KVCache, k.to(S8), k.to(S8), torch.zeros(4, 16, 2), torch.zeros(4, 2, 16))
    refused(INVALID, api.KVCache, k.to(S8), k.to(S8), torch.zeros(4, 16, 2, dtype=F16), torch.zeros(4, 16, 2, dtype=F16))
    n = torch.zeros(1, dtype=torch.int64)
    for dtype, dim, code in ((BF16, 136, UNSUPPORTED), (BF16, 12, UNSUPPORTED), (S8, 72, UNSUPPORTED), (F32, 64, INVALID), (torch.uint8, 64, INVALID)):
        c = cache(dtype, dim=dim)
        refused(code, api.pulpnn_kv_append, c, n, rows(1, 2, dim, F32), rows(1, 2, dim, F32))
    raw = torch.zeros(4 * 16 * 2 * 64 + 4, dtype=BF16)
    odd = raw[4:].view(4, 16, 2, 64)                       # 8 bytes off a 16-byte boundary
    if raw.data_ptr() % 16 == 0:
        refused(UNSUPPORTED, api.pulpnn_kv_append, api.KVCache(odd, odd), n, rows(1, 2, 64), rows(1, 2, 64))
    pitched = torch.zeros(4, 16, 2, 68, dtype=BF16)[..., :64]
    refused(UNSUPPORTED, api.pulpnn_kv_append, api.KVCache(pitched, pitched), n, rows(1, 2, 64), rows(1, 2, 64))


def test_append():
    c, n, k = cache(), torch.arange(3), rows(3, 2, 64)
    call = api.pulpnn_kv_append
    refused(INVALID, call, c, n, rows(3, 3, 64), k)
    refused(INVALID, call, c, n, k, rows(2, 2, 64))
    refused(INVALID, call, c, n, k, k.to(F16))
    refused(INVALID, call, c, n.to(S32), k, k)
    refused(INVALID, call, c, n[:2], k, k)
    refused(INVALID, call, c, n, k, k, q=rows(3, 4, 64))
    refused(INVALID, call, c, n, k, k, q=rows(3, 4, 64), q_out=rows(3, 4, 64, F32))
    refused(INVALID, call, c, n, k, k, q=rows(3, 4, 64), q_out=rows(3, 4, 64, F16), k_out=k)
    refused(INVALID, call, c, n, k, k, q=rows(3, 4, 64), q_out=rows(1, 4, 64).expand(3, 4, 64))
    refused(INVALID, call, c, n, k, k, inv_freq=torch.ones(32, dtype=torch.float64))
    refused(INVALID, call, c, n, k, k, inv_freq=torch.ones(32), positions=n.to(S32))
    refused(INVALID, call, c, n, k, k, inv_freq=torch.ones(33, dtype=torch.float64), positions=n.to(S32))
    refused(INVALID, call, c, n, k, k, k_step=torch.ones(128))
    refused(INVALID, call, c, n, k.to(S32), k.to(S32))
    refused(INVALID, call, c, n, k.to(S32), k.to(S32), k_step=torch.ones(64), v_step=torch.ones(128))
    refused(INVALID, call, c, n, k.to(S8), k.to(S8))
    refused(UNSUPPORTED, call, c, n, torch.zeros(3, 2, 68, dtype=BF16)[..., :64], k)
    refused(INVALID, call, c, n, torch.zeros(3, 2, 128, dtype=BF16)[..., ::2], k)
    call(c, n[:0], k[:0], k[:0])                            # nothing to do


def test_gather():
    c, n = cache(), torch.arange(3)
    refused(INVALID, api.pulpnn_kv_gather, c, n, None, None)
    refused(INVALID, api.pulpnn_kv_gather, c, n, rows(2, 2, 64))
    refused(INVALID, api.pulpnn_kv_gather, c, n, rows(3, 2, 64), rows(3, 2, 64, F16))
    refused(UNSUPPORTED, api.pulpnn_kv_gather, c, n, rows(3, 2, 64, F16))
    refused(INVALID, api.pulpnn_kv_gather, c, n, rows(3, 2, 64, F32))
    api.pulpnn_kv_gather(c, n[:0], rows(0, 2, 64))


def test_decode():
    c, q, table, lens = cache(), rows(3, 4, 64), torch.zeros(3, 2, dtype=S32), torch.zeros(3, dtype=S32)
    call = api.pulpnn_attn_decode
    refused(INVALID, call, c, q[..., :32], table, lens, q)
    refused(INVALID, call, c, q, table, lens, q[:2])
    refused(INVALID, call, c, q, table[:2], lens, q)
    refused(INVALID, call, c, q, table.long(), lens, q)
    refused(INVALID, call, c, q, table, lens.long(), q)
    refused(INVALID, call, c, q, torch.zeros(3, 4, dtype=S32)[:, ::2], lens, q)
    refused(INVALID, call, c, q, table, lens, q.to(F16))
    refused(INVALID, call, c, q, table, lens, q.to(torch.uint8))
    refused(INVALID, call, c, q, table, lens, q, out_step=0.1)
    refused(INVALID, call, c, q, table, lens, q.to(torch.uint8), out_step=0.1, out_zero=256)
    refused(INVALID, call, c, q, table, lens, q.to(torch.uint8), out_step=-0.1)
    refused(UNSUPPORTED, call, c, q.to(F16), table, lens, q.to(F16))
    refused(INVALID, call, c, q[:, :3], table, lens, q[:, :3].clone())
    refused(INVALID, call, c, q, table, lens, q, window=-1)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(INVALID, call, c, q, table, lens, q, scale=scale)
    refused(INVALID, call, c, q, table, lens, q, lse=torch.zeros(3, 5))
    refused(INVALID, call, c, q, table, lens, q, lse=torch.zeros(3, 4, dtype=F16))
    call(c, q[:0], table[:0], lens[:0], q[:0])


def test_decode_of_tables_for_2_31_tokens():
    # 524273 pages of 4096 slots: 2^31 - 61440 tokens, which a few tiles more would carry beyond 31 bits
    c, q = cache(pages=1, page=4096, heads=1, dim=8), rows(1, 1, 8)
    refused(UNSUPPORTED, api.pulpnn_attn_decode, c, q, torch.zeros(1, 524273, dtype=S32), torch.zeros(1, dtype=S32), q.clone())


def test_prompt():
    q, k, cu = rows(7, 4, 64), rows(7, 2, 64), torch.tensor([0, 7], dtype=S32)
    call = api.pulpnn_attn_prompt
    refused(INVALID, call, q, k, k[:6], cu, q)
    refused(INVALID, call, q, k[:6], k[:6], cu, q)
    refused(INVALID, call, q, k, k.to(F16), cu, q)
    refused(UNSUPPORTED, call, q.float(), k.float(), k.float(), cu, q.float())
    refused(INVALID, call, q, rows(7, 3, 64), rows(7, 3, 64), cu, q.clone())
    refused(INVALID, call, q, k, k, cu.long(), q)
    refused(INVALID, call, q, k, k, cu, q, cu_k=torch.zeros(3, dtype=S32))
    refused(INVALID, call, q, k, k, cu, q, window=3, causal=False)
    refused(INVALID, call, q, k, k, cu, q, window=-3)
    refused(INVALID, call, q, k, k, cu, q, scale=0.0)
    refused(INVALID, call, q, k, k, cu, q, out_step=1.0)
    refused(INVALID, call, q, k, k, cu, q.to(torch.uint8), out_step=0.0)
    refused(INVALID, call, q, k, k, cu, q[:, :1].expand(7, 4, 64))
    refused(UNSUPPORTED, call, q, k[:, :1].expand(7, 2, 64), k, cu, q.clone())
    refused(UNSUPPORTED, call, rows(7, 4, 136), rows(7, 2, 136), rows(7, 2, 136), cu, rows(7, 4, 136))
    refused(UNSUPPORTED, call, rows(7, 4, 12), rows(7, 2, 12), rows(7, 2, 12), cu, rows(7, 4, 12))
    call(q[:0], k[:0], k[:0], cu, q[:0])
    call(q, k, k, cu[:1], q)                               # no sequences


def test_null_structs():
    lib = pulpnn.load_library()
    for name, n in (("pulpnn_kv_append", 2), ("pulpnn_kv_gather", 2), ("pulpnn_attn_decode", 2), ("pulpnn_attn_prompt", 1)):
        f = getattr(lib, name)
        f.restype, f.argtypes = C.c_int, [C.c_char_p] * n
        assert f(*[None] * n) == INVALID
        lib.pulpnn_clear_error()


@pytest.mark.skipif(_has_gpu(), reason="checks the behaviour on a machine without a GPU")
def test_no_gpu_is_an_error():
    q, k, cu = rows(7, 4, 64), rows(7, 2, 64), torch.tensor([0, 7], dtype=S32)
    refused(api.ERR_NO_DEVICE, api.pulpnn_attn_prompt, q, k, k, cu, q.clone())
    refused(api.ERR_NO_DEVICE, api.pulpnn_kv_append, cache(), torch.arange(7), k, k)


@pytest.mark.gpu
def test_host_memory_is_refused():
    pulpnn.GpuKernels()
    q, k, cu = rows(7, 4, 64), rows(7, 2, 64), torch.tensor([0, 7], dtype=S32)
    gpu = [t.cuda() for t in (q, k, k, cu, q)]
    for i in range(5):
        a = list(gpu)
        a[i] = (q, k, k, cu, q)[i]
        refused(INVALID, api.pulpnn_attn_prompt, *a)
        a[i] = a[i].pin_memory()
        refused(INVALID, api.pulpnn_attn_prompt, *a)
    refused(INVALID, api.pulpnn_kv_append, cache(), torch.arange(7).cuda(), gpu[1], gpu[1])
    c = torch.zeros(4, 16, 2, 64, dtype=BF16, device="cuda")
    handle = api.KVCache(c, c.clone())
    refused(INVALID, api.pulpnn_kv_append, handle, torch.arange(7), gpu[1], gpu[1])
    refused(INVALID, api.pulpnn_kv_gather, handle, torch.arange(7).cuda(), k)
    refused(INVALID, api.pulpnn_attn_decode, handle, gpu[0], torch.zeros(7, 1, dtype=S32), torch.zeros(7, dtype=S32).cuda(), gpu[4])
