"""Attention over a paged cache where it is easily wrong: work without keys, values at the ends of the types, rarely taken paths."""
import math
import threading
from types import SimpleNamespace

import pytest

from conftest import pulpnn

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from attention_cases import Fenced, attend, eps, tolerance  # noqa: E402
from test_gpu_attention import BF16, F16, S8, Cache, _settled, freqs, gen, normal, prompt_case  # noqa: E402, F401

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


# ---- rows of 8 bits ----------------------------------------------------------------------------------------

def test_append_writes_rows_that_8_bits_cannot_hold_as_they_are():
    """k_out and v_out get a row before it is cut to 8 bits: infinities, NaN and the smallest values among them."""
    g = gen(26)
    x = normal(g, 6, 2, 64)
    x[1] = 0
    x[2] *= 1e-36
    x[3, 0, 5], x[3, 1, 6] = math.inf, -math.inf
    x[4, 0, 63] = math.nan
    c = Cache(g, S8, 1, 8, 2, 64, False)
    outs = [torch.empty(6, 2, 64, dtype=BF16, device="cuda") for _ in range(2)]
    api.pulpnn_kv_append(c.handle, torch.arange(6, device="cuda"), x, -x, k_out=outs[0], v_out=outs[1])
    torch.cuda.synchronize()
    for out, want in zip(outs, (x, -x)):
        torch.testing.assert_close(out, want.to(BF16), rtol=0, atol=0, equal_nan=True)


# ---- append in place ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim,rot,interleaved", [(112, 20, False), (128, 126, False), (80, 32, False), (128, 128, False), (80, 32, True), (48, 14, True),
                                                 (72, 72, False), (72, 70, False)])
def test_append_in_place_is_append(dtype, dim, rot, interleaved):
    """Every way the rotation takes its pairs, several batches of rows a warp: the same bits as in buffers of their own."""
    g = gen(rot)
    n, hq, hkv = 700, 37, 9
    c = [Cache(gen(1), dtype, 50, 16, hkv, dim, False) for _ in range(2)]
    slots = torch.randperm(800, generator=g, device="cuda")[:n]
    pos = torch.randint(0, 100000, (n,), generator=g, device="cuda").to(torch.int32)
    packed = normal(g, n, hq + 2 * hkv, dim, dtype=dtype)
    cut = lambda x: (x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:])  # noqa: E731
    out = torch.empty_like(packed)
    (q, k, v), (qo, ko, vo) = cut(packed), cut(out)
    api.pulpnn_kv_append(c[0].handle, slots, k, v, positions=pos, inv_freq=freqs(rot), interleaved=interleaved, q=q, q_out=qo, k_out=ko, v_out=vo)
    api.pulpnn_kv_append(c[1].handle, slots, k, v, positions=pos, inv_freq=freqs(rot), interleaved=interleaved, q=q, q_out=q, k_out=k, v_out=v)
    torch.cuda.synchronize()
    assert torch.equal(packed, out)
    at = torch.arange(800, device="cuda")
    assert all(torch.equal(c[0].rows(i, at), c[1].rows(i, at)) for i in range(2))


# ---- strides that go backwards (the C interface has them; torch does not) ------------------------------------

@pytest.mark.parametrize("dtype", [BF16, S8])
def test_caches_and_rows_at_negative_strides(dtype):
    g = gen(27)
    pages, page, hkv, dim = 5, 16, 3, 64
    c = Cache(g, dtype, pages, page, hkv, dim, False)
    kept = [x.wide for x in (c.k, c.v)] + ([x.wide for x in c.s] if c.s else [])
    before = [t.clone() for t in kept]
    # the same memory with its pages, slots and heads counted from the last
    flip = lambda x: sum((n - 1) * s for n, s in zip(x.shape[:3], x.stride()[:3])) * x.element_size()  # noqa: E731
    s = [t.view for t in c.s] if c.s else [None, None]
    base = [t.data_ptr() + flip(t) if t is not None else 0 for t in (c.k.view, c.v.view, *s)]
    a, b = c.k.view.stride(), s[0].stride() if c.s else (0, 0, 0)
    block = api.KVCache._pack(*base, -a[0], -a[1], -a[2], -b[0], -b[1], -b[2], c.handle.type, pages, page, hkv, dim, 0)
    back = SimpleNamespace(block=block, type=c.handle.type, n_pages=pages, page_size=page, n_heads=hkv, head_dim=dim)
    n = 40
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:n]
    mirrored = pages * page - 1 - slots
    k, v = normal(g, n, hkv, dim, dtype=BF16), normal(g, n, hkv, dim, dtype=BF16)
    api.pulpnn_kv_append(c.handle, mirrored, k.flip(1).contiguous(), v.flip(1).contiguous())
    torch.cuda.synchronize()
    want = [t.clone() for t in kept]
    for t, old in zip(kept, before):
        t.copy_(old)
    api.pulpnn_kv_append(back, slots, k, v)
    torch.cuda.synchronize()
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(kept, want)) and c.intact()
    # read back, into rows whose tokens and heads go backwards
    straight, turned = ([Fenced((n, hkv, dim), BF16) for _ in range(2)] for _ in range(2))
    api.pulpnn_kv_gather(back, slots, straight[0].view, straight[1].view)
    o = [x.view for x in turned]
    api._gather_call(block, api._gather_pack(slots.data_ptr(), *(x[-1, -1].data_ptr() for x in o), *[-o[0].stride(0), -o[0].stride(1)] * 2, n, api.TYPE_BF16))
    torch.cuda.synchronize()
    for i in range(2):
        assert straight[i].intact() and turned[i].intact()
        stored = c.rows(i, mirrored).flip(1)
        assert ((straight[i].view.double() - stored).abs() <= (eps(BF16) / 2 + 2.0 ** -23) * stored.abs()).all()
        assert torch.equal(o[i].flip(0, 1), straight[i].view)
    # one token reads the same cache
    q, lens = normal(g, 1, 6, dim, dtype=BF16), torch.tensor([pages * page], dtype=torch.int32, device="cuda")
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    out = torch.empty_like(q)
    api.pulpnn_attn_decode(back, q, table, lens, out)
    torch.cuda.synchronize()
    at = torch.arange(pages * page - 1, -1, -1, device="cuda")
    kk, vv = (c.rows(i, at).flip(1) for i in range(2))
    for h in range(6):
        w, _, sums, product = attend(q[0, h:h + 1].double(), kk[:, h // 2], vv[:, h // 2], torch.ones(1, len(at), dtype=torch.bool, device="cuda"), dim ** -0.5)
        assert ((out[0, h].double() - w[0]).abs() <= tolerance(w, sums, product, len(at), dim, BF16, F16 if dtype == S8 else BF16)[0]).all()


# ---- scores and weights at the ends of the types ----------------------------------------------------------

def one_sequence(cache_type, k, v, page=16, k_scale=1.0, v_scale=1.0):
    """A cache of one sequence's rows ([n][dim] each), in order, with its table."""
    n, dim = k.shape
    pages = -(-n // page)
    rows = [torch.zeros(pages * page, dim, dtype=cache_type, device="cuda") for _ in range(2)]
    for r, x in zip(rows, (k, v)):
        r[:n] = x.to(cache_type)
    scales = [None, None]
    if cache_type == S8:
        scales = [torch.zeros(pages * page, device="cuda") for _ in range(2)]
        for s, x in zip(scales, (k_scale, v_scale)):
            s[:n] = x
        scales = [s.view(pages, page, 1) for s in scales]
    cache = api.KVCache(*(r.view(pages, page, 1, dim) for r in rows), *scales)
    return cache, torch.arange(pages, dtype=torch.int32, device="cuda")[None], torch.tensor([n], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("how", ["decode", "decode s8", "prompt 64", "prompt 128"])
def test_many_small_weights_beside_a_large_one(how):
    """4095 weights of 2^-27 of the largest one each. In fp16, which holds nothing below 2^-24, they must not vanish from the sum over
    the values: the largest weight is held at 2^5 or more, and each of the small ones is then off by 2^-25 at most."""
    n, dim = 4096, 128 if how == "prompt 128" else 64
    q, k, v = torch.zeros(1, 1, dim, device="cuda"), torch.zeros(n, dim, device="cuda"), torch.zeros(n, dim, device="cuda")
    q[..., 0] = 8
    k[0, 0], v[1:] = 117 / 50, 1016.0
    out = torch.empty(1, 1, dim, dtype=F16, device="cuda")
    lse = torch.empty(1, 1, device="cuda")
    if how.startswith("decode"):
        eight = how.endswith("s8")
        cache = one_sequence(S8, k * 50, v / 8, k_scale=0.02, v_scale=8.0) if eight else one_sequence(F16, k, v)
        kept = (k * 50).to(S8).double() * float(torch.tensor(0.02)) if eight else k.to(F16)      # as it lies in the cache
        api.set_option(api.OPT_SPLIT_K, 1)
        try:
            api.pulpnn_attn_decode(cache[0], q.to(F16), cache[1], cache[2], out, scale=1.0, lse=lse)
        finally:
            api.set_option(api.OPT_SPLIT_K, 0)
    else:
        cu_q, cu_k = (torch.tensor([0, m], dtype=torch.int32, device="cuda") for m in (1, n))
        kept = k.to(F16)
        api.pulpnn_attn_prompt(q.to(F16), kept[:, None], v.to(F16)[:, None], cu_q, out, cu_k=cu_k, scale=1.0, lse=lse)
    torch.cuda.synchronize()
    score = 8 * kept[0, 0].double()
    small = (n - 1) * (-score).exp()
    want = 1016 * small / (1 + small)
    # rounded to fp16 once; each small weight by half of fp16's smallest step where the largest is 2^5; sums and exponents in 32 bits
    tol = eps(F16) / 2 * want + n * 2.0 ** -25 * 2.0 ** -5 * 1016 + 2.0 ** -16 * want
    assert ((out.double() - want).abs() <= tol).all(), (out[0, 0, 0], want)
    assert abs(lse.double() - (score + torch.log1p(small))) <= 2.0 ** -16


@pytest.mark.parametrize("how", ["decode", "decode s8", "decode window", "prompt 64", "prompt 128"])
def test_scores_of_a_large_negative_number(how):
    """Scores of about -10^37, all equal: an average of the values, and not the zeros of a row without keys."""
    n, dim = 300, 128 if how == "prompt 128" else 64
    g = gen(28)
    q, k = torch.full((1, 1, dim), -2.0 ** 60, device="cuda", dtype=BF16), torch.full((n, dim), 2.0 ** 60, device="cuda", dtype=BF16)
    v = torch.randint(-100, 100, (n, dim), generator=g, device="cuda").to(BF16)
    out, lse = torch.empty(1, 1, dim, dtype=BF16, device="cuda"), torch.empty(1, 1, device="cuda")
    window = 130 if how == "decode window" else 0
    if how.startswith("decode"):
        cache = one_sequence(S8, torch.full_like(k, 64), v, k_scale=2.0 ** 54) if how.endswith("s8") else one_sequence(BF16, k, v)
        api.pulpnn_attn_decode(cache[0], q, cache[1], cache[2], out, lse=lse, window=window)
    else:
        cu_q, cu_k = (torch.tensor([0, m], dtype=torch.int32, device="cuda") for m in (1, n))
        api.pulpnn_attn_prompt(q, k[:, None], v[:, None], cu_q, out, cu_k=cu_k, lse=lse)
    torch.cuda.synchronize()
    seen = v[-window:].double()
    want = seen.mean(0)
    # equal weights of one: their sum and the products are whole numbers; divided in 32 bits, rounded to bf16 once
    assert ((out[0, 0].double() - want).abs() <= (eps(BF16) / 2 + 2.0 ** -20) * want.abs()).all()
    score = -2.0 ** 120 * dim * dim ** -0.5
    assert abs(lse[0, 0].double() / score - 1) <= (dim + 8) * 2.0 ** -23


@pytest.mark.parametrize("dtype,u,w", [(F16, 1.0, 64.0), (BF16, 2.0 ** 17, 2.0 ** 30)])
@pytest.mark.parametrize("how", ["decode", "prompt 64", "prompt 128"])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_far_apart(how, dtype, u, w, sign):
    """Scores of up to 2^33 and 2^75, far apart: the value of the largest one, or the mean of two where it comes twice."""
    n, dim, rows = 300, 128 if how == "prompt 128" else 64, 12
    g = gen(31)
    order = (torch.randperm(n, generator=g, device="cuda") % 250 + 1).float()        # the largest one once, the smallest ones twice
    k = (order[:, None].expand(n, dim) * w).to(dtype)
    q = (torch.tensor([sign * m for m in (3, 37, 513, 1025, 1027, 4099, 8199, 10001, 12347, 20011, 30011, 31013)], device="cuda")[:, None, None].expand(rows, 1, dim) * u).to(dtype)
    v = torch.randint(-100, 100, (n, dim), generator=g, device="cuda").to(dtype)
    out = torch.empty(rows, 1, dim, dtype=dtype, device="cuda")
    if how == "decode":
        cache = one_sequence(dtype, k, v)
        api.pulpnn_attn_decode(cache[0], q, cache[1].expand(rows, -1).contiguous(), cache[2].expand(rows).contiguous(), out)
    else:
        cu_q, cu_k = (torch.tensor([0, m], dtype=torch.int32, device="cuda") for m in (rows, n))
        api.pulpnn_attn_prompt(q.contiguous(), k[:, None].contiguous(), v[:, None], cu_q, out, cu_k=cu_k, causal=False)
    torch.cuda.synchronize()
    x = sign * k[:, 0].double()
    best = x == x.max()
    # the next score is at least 3 x 64 / 8 below: e^-24 of a value of up to 100, which a result of 0 shows by itself
    want = v[best].double().mean(0)
    assert ((out[:, 0].double() - want).abs() <= eps(dtype) / 2 * want.abs() + 300 * 100 * math.exp(-24)).all()


@pytest.mark.parametrize("top", [126, 127])
def test_decode_8_bits_with_queries_at_the_end_of_bf16(top):
    """Queries of up to 2^127 on keys of 2^-126: scores that are ordinary numbers."""
    g = gen(top)
    n, dim, hq = 100, 64, 2
    q = normal(g, 1, hq, dim) * 2.0 ** 120
    q[..., 3], q[..., 9] = 2.0 ** top, -1.5 * 2.0 ** top
    q = q.to(BF16)
    codes = torch.randint(-127, 128, (2, n, dim), generator=g, device="cuda")
    cache = one_sequence(S8, codes[0], codes[1], k_scale=2.0 ** -126, v_scale=0.01)
    out = torch.empty_like(q)
    api.pulpnn_attn_decode(cache[0], q, cache[1], cache[2], out)
    torch.cuda.synchronize()
    k, v = codes[0].double() * 2.0 ** -126, codes[1].double() * float(torch.tensor(0.01))
    want, _, sums, product = attend(q[0].double(), k, v, torch.ones(hq, n, dtype=torch.bool, device="cuda"), dim ** -0.5)
    # a key's product with q, scaled to a largest value of 1 .. 2, may fall below 2^-126 times its scale: off by 2^-149 x 2^127 there
    assert ((out[0].double() - want).abs() <= tolerance(want, sums, product + 1, n, dim, BF16, F16)).all()


def test_decode_8_bits_rows_of_zeros_whatever_their_scale():
    """A row of codes of zero has the score 0, also where its scale times the query's size is beyond 32 bits."""
    g = gen(29)
    n, dim = 100, 64
    q = (normal(g, 1, 2, dim) * 2.0 ** 100).to(BF16)
    codes = torch.randint(-127, 128, (2, n, dim), generator=g, device="cuda")
    codes[0, ::3] = 0
    scale = torch.full((n,), 2.0 ** -104, device="cuda")
    scale[::3] = 2.0 ** 40
    cache = one_sequence(S8, codes[0], codes[1], k_scale=scale, v_scale=0.01)
    out = torch.empty_like(q)
    api.pulpnn_attn_decode(cache[0], q, cache[1], cache[2], out)
    torch.cuda.synchronize()
    k, v = codes[0].double() * scale.double()[:, None], codes[1].double() * float(torch.tensor(0.01))
    want, _, sums, product = attend(q[0].double(), k, v, torch.ones(2, n, dtype=torch.bool, device="cuda"), dim ** -0.5)
    assert ((out[0].double() - want).abs() <= tolerance(want, sums, product + 1, n, dim, BF16, F16)).all()


# ---- beside a capture of another thread -----------------------------------------------------------------------

@pytest.mark.parametrize("first", ["decode", "prompt"])
def test_a_threads_first_call_beside_a_capture_of_another(first):
    """A thread's first attention, which gets the word its waits report into, while another thread captures a graph."""
    g = gen(30)
    p = normal(g, 40, 4, 64, dtype=BF16)
    cu, out = torch.tensor([0, 40], dtype=torch.int32, device="cuda"), torch.empty_like(p)
    c = Cache(g, BF16, 4, 16, 2, 64, False)
    table, lens = torch.arange(3, dtype=torch.int32, device="cuda")[None], torch.tensor([40], dtype=torch.int32, device="cuda")
    mark = torch.ones(8, device="cuda")

    def call():
        if first == "decode":
            api.pulpnn_attn_decode(c.handle, p[:1], table, lens, out[:1])
        else:
            api.pulpnn_attn_prompt(p, p[:, :2], p[:, 2:], cu, out)

    call()                                                   # loads the kernel
    torch.cuda.synchronize()
    want, errors = out.clone(), []
    out.zero_()

    def work():
        try:
            torch.cuda.set_device(0)
            api.set_device(0)
            api.set_stream(stream)
            ready.set()
            capturing.wait(60)
            call()
        except BaseException as e:
            errors.append(e)

    ready, capturing = threading.Event(), threading.Event()
    stream, side, graph = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    t = threading.Thread(target=work)
    t.start()
    assert ready.wait(60)
    with torch.cuda.graph(graph, stream=side):
        mark.zero_()
        capturing.set()
        t.join()
    graph.replay()
    torch.cuda.synchronize()
    assert not errors, errors
    rows = slice(0, 1) if first == "decode" else slice(None)
    assert not mark.any() and torch.equal(out[rows], want[rows])


# ---- what is masked, beside rarely taken paths ------------------------------------------------------------------

@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (BF16, 80)])
def test_prompt_infinities_and_uint8_output(dtype, dim):
    """Infinities in V that some rows of a tile see and others do not, and an output of uint8: 255 and 0 for those that do, the
    zero point for infinities of both signs together, what the finite values give for the others."""
    g = gen(32)
    n, step, zero = 200, 0.02, 100
    q, k, v = (normal(g, n, 1, dim, dtype=dtype) for _ in range(3))
    v[150, 0, ::2], v[170, 0, 1::2], v[190, 0, 0] = math.inf, -math.inf, -math.inf
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    out = torch.empty(n, 1, dim, dtype=torch.uint8, device="cuda")
    api.pulpnn_attn_prompt(q, k, v, cu, out, out_step=step, out_zero=zero)
    torch.cuda.synchronize()
    finite = v[:, 0].double().where(v[:, 0].isfinite(), torch.zeros_like(v[:, 0], dtype=torch.float64))
    seen = torch.tril(torch.ones(n, n, dtype=torch.bool, device="cuda"))
    want, _, sums, product = attend(q[:, 0].double(), k[:, 0].double(), finite, seen, dim ** -0.5)
    tol = tolerance(want, sums, product, n, dim, None, dtype) / step
    got, want = out[:, 0].double(), (want / step + zero).clamp(0, 255)
    row, channel = torch.arange(n, device="cuda")[:, None], torch.arange(dim, device="cuda")[None]
    up, down = (row >= 150) & (channel % 2 == 0), (row >= 170) & (channel % 2 == 1)
    both = (row >= 190) & (channel == 0)
    assert (got[up & ~both] == 255).all() and (got[down] == 0).all() and (got[both] == zero).all()
    assert ((got - want).abs() <= 0.5 + tol + 1e-4)[~up & ~down].all()
