"""Attention over a paged cache of keys and values against its definition in 64 bits."""
import math

import numpy as np
import pytest

from conftest import pulpnn

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from attention_cases import Fenced, attend, eps, lse_tolerance, rotate, tolerance  # noqa: E402

api = pulpnn.api
F16, BF16, F32, S32, S8 = torch.float16, torch.bfloat16, torch.float32, torch.int32, torch.int8


@pytest.fixture(autouse=True)
def _settled():
    pulpnn.GpuKernels()
    api.set_stream(None)
    yield
    torch.cuda.synchronize()
    assert api.device_status() == 0


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


class Cache:
    """A fenced cache with its handle, and its rows in 64 bits."""

    def __init__(self, g, dtype, pages, page, heads, dim, heads_first, fill=True):
        shape = (pages, heads, page) if heads_first else (pages, page, heads)
        self.page, self.heads_first, self.dtype = page, heads_first, dtype
        self.k, self.v = Fenced(shape + (dim,), dtype), Fenced(shape + (dim,), dtype)
        self.s = None
        if dtype == S8:
            self.s = [Fenced(shape, F32), Fenced(shape, F32)]
        for i, x in enumerate((self.k, self.v)):
            if not fill:
                x.view.zero_()
            elif dtype == S8:
                x.view.copy_(torch.randint(-127, 128, shape + (dim,), generator=g, device="cuda"))
            else:
                x.view.copy_(normal(g, *shape, dim))
            if self.s:
                self.s[i].view.copy_(torch.rand(shape, generator=g, device="cuda") * 0.02 + 0.005 if fill else torch.zeros(shape))
        s = [None, None] if self.s is None else [x.view for x in self.s]
        self.handle = api.KVCache(self.k.view, self.v.view, s[0], s[1], heads_first=heads_first)

    def rows(self, which, slots):
        x = (self.k, self.v)[which].view
        x = x.transpose(1, 2) if self.heads_first else x
        r = x[slots // self.page, slots % self.page].double()
        if self.s is not None:
            s = self.s[which].view
            s = s.transpose(1, 2) if self.heads_first else s
            r = r * s[slots // self.page, slots % self.page].double()[..., None]
        return r

    def intact(self):
        return self.k.intact() and self.v.intact() and (self.s is None or all(x.intact() for x in self.s))


def freqs(rot):
    return None if not rot else 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)


# ---- append and gather --------------------------------------------------------------------------------

@pytest.mark.parametrize("in_type,wide,cache", [(BF16, BF16, BF16), (F16, F16, S8), (F32, F16, F16), (S32, BF16, S8), (BF16, BF16, S8),
                                                (S32, F16, F16), (F32, BF16, S8), (S32, BF16, F16), (BF16, F16, BF16)])
@pytest.mark.parametrize("n,hq,hkv,dim,rot,interleaved,heads_first,page", [
    (1, 4, 1, 128, 128, False, False, 16), (37, 3, 3, 80, 32, True, True, 20), (5, 7, 1, 64, 64, False, True, 1),
    (19, 2, 2, 112, 20, False, False, 7), (9, 1, 1, 16, 10, True, False, 16), (700, 4, 2, 32, 0, False, False, 33),
    (3, 33, 2, 128, 126, False, False, 16), (5003, 5, 1, 32, 32, False, True, 64), (3001, 2, 3, 48, 14, True, False, 20)])
def test_append(in_type, wide, cache, n, hq, hkv, dim, rot, interleaved, heads_first, page):
    g = gen(n * 131 + dim)
    pages = (n + 5) // page + 2
    c = Cache(g, cache, pages, page, hkv, dim, heads_first, fill=True)
    before = [c.rows(i, torch.arange(pages * page, device="cuda")) for i in range(2)]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:n].clone()
    if n > 3:
        slots[1], slots[2], slots[3] = -1, pages * page, 2 ** 40
    positions = torch.randint(0, 200000, (n,), generator=g, device="cuda").to(torch.int32)
    x, step = {}, {}
    for name, heads in (("q", hq), ("k", hkv), ("v", hkv)):
        if in_type == S32:
            x[name] = Fenced((n, heads, dim), S32, fill=torch.randint(-2 ** 20, 2 ** 20, (n, heads, dim), generator=g, device="cuda"))
            step[name] = torch.rand(heads * dim, generator=g, device="cuda") * 1e-5
        else:
            x[name] = Fenced((n, heads, dim), in_type, fill=normal(g, n, heads, dim))
            step[name] = None
    out = {name: Fenced((n, heads, dim), wide) for name, heads in (("q", hq), ("k", hkv), ("v", hkv))}
    api.pulpnn_kv_append(c.handle, slots, x["k"].view, x["v"].view, positions=positions, inv_freq=freqs(rot), interleaved=interleaved,
                         q=x["q"].view, q_out=out["q"].view, k_out=out["k"].view, v_out=out["v"].view, q_step=step["q"],
                         k_step=step["k"], v_step=step["v"])
    torch.cuda.synchronize()
    assert api.last_kernel() == "kv_append_kernel"
    assert c.intact() and all(o.intact() for o in out.values())
    stored = (slots >= 0) & (slots < pages * page)
    for i, name in enumerate(("q", "k", "v")):
        raw = x[name].view.double()
        if step[name] is not None:
            raw = raw * step[name].double().view(1, -1, dim)
        want = raw if name == "v" else rotate(raw, positions, freqs(rot), interleaved)
        # in 32 bits: a product by the step, two products and a sum, and sines off by 2^-22 (their argument, below pi, by 2^-24 of it)
        size = raw.abs()
        if rot and name != "v":
            half = rot // 2
            a, b = (size[..., 0:rot:2], size[..., 1:rot:2]) if interleaved else (size[..., :half], size[..., half:rot])
            both = a + b
            size = size.clone()
            if interleaved:
                size[..., 0:rot:2], size[..., 1:rot:2] = both, both
            else:
                size[..., :half], size[..., half:rot] = both, both
        off = 2.0 ** -20 * size
        err = (out[name].view.double() - want).abs()
        assert (err <= eps(wide) / 2 * want.abs() + off * 1.01 + torch.finfo(wide).smallest_normal * eps(wide)).all(), name
        if name == "q":
            continue
        got = c.rows(i - 1, slots[stored])
        err = (got - want[stored]).abs()
        if cache == S8:
            # half a code, and the code's and the scale's own 32-bit errors
            most = want[stored].abs().amax(-1, keepdim=True)
            bound = most / 127 * 0.5 + (off[stored].amax(-1, keepdim=True) + most * 2.0 ** -20) * 2
        else:
            bound = eps(cache) / 2 * want[stored].abs() + off[stored] * 1.01 + torch.finfo(cache).smallest_normal * eps(cache)
        assert (err <= bound).all(), name
        rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
        rest[slots[stored]] = False
        now = c.rows(i - 1, torch.arange(pages * page, device="cuda"))
        assert torch.equal(now[rest], before[i - 1][rest])


@pytest.mark.parametrize("in_type,wide,cache", [(BF16, BF16, BF16), (S32, F16, F16)])
@pytest.mark.parametrize("dim,rot,interleaved", [(72, 72, False), (72, 72, True), (72, 24, True), (8, 8, False), (8, 0, False), (104, 2, True), (24, 16, False)])
def test_append_an_odd_number_of_octets(in_type, wide, cache, dim, rot, interleaved):
    test_append(in_type, wide, cache, 37, 3, 2, dim, rot, interleaved, True, 5)


def test_append_in_place_and_without_queries():
    g = gen(3)
    n, hkv, dim = 23, 4, 96
    c = Cache(g, BF16, 3, 16, hkv, dim, False, fill=False)
    packed = Fenced((n, 12, dim), BF16, fill=normal(g, n, 12, dim))          # q, k and v of a token side by side
    q, k, v = packed.view[:, :4], packed.view[:, 4:8], packed.view[:, 8:]
    q0, k0, v0 = (t.double().clone() for t in (q, k, v))
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    slots = torch.arange(n, device="cuda")
    api.pulpnn_kv_append(c.handle, slots, k, v, positions=pos, inv_freq=freqs(96), q=q, q_out=q, k_out=k, v_out=v)
    torch.cuda.synchronize()
    assert packed.intact() and torch.equal(v.double(), v0)
    for got, raw in ((q, q0), (k, k0), (c.rows(0, slots), k0)):
        want = rotate(raw, pos, freqs(96), False)
        assert ((got.double() - want).abs() <= eps(BF16) / 2 * want.abs() + 2.0 ** -19 * raw.abs().amax()).all()
    k1 = normal(g, n, hkv, dim, dtype=BF16)
    api.pulpnn_kv_append(c.handle, slots, k1, v)                              # no rotation, no queries
    torch.cuda.synchronize()
    assert torch.equal(c.rows(0, slots), k1.double())


def test_append_and_gather_with_strides_beyond_32_bits():
    """Tokens 1 GB apart, in what is read and in what is written."""
    g = gen(16)
    n, far = 5, 2 ** 29
    wide = torch.empty(n * far, dtype=BF16, device="cuda")
    view = lambda at: wide[at:].as_strided((n, 2, 64), (far, 64, 1))  # noqa: E731
    q, k, v, k_out = (view(at) for at in (0, 256, 512, 768))
    for t in (q, k, v):
        t.copy_(normal(g, n, 2, 64))
    q0, k0, v0 = (t.double().clone() for t in (q, k, v))
    pos = torch.arange(n, device="cuda", dtype=torch.int32) + 70000
    slots = torch.arange(n, device="cuda") + 3
    c = Cache(g, BF16, 1, 8, 2, 64, False)
    api.pulpnn_kv_append(c.handle, slots, k, v, positions=pos, inv_freq=freqs(64), q=q, q_out=q)
    api.pulpnn_kv_gather(c.handle, slots, k_out)
    torch.cuda.synchronize()
    for got, raw in ((q, q0), (k_out, k0), (c.rows(0, slots), k0)):
        want = rotate(raw, pos, freqs(64), False)
        assert ((got.double() - want).abs() <= eps(BF16) / 2 * want.abs() + 2.0 ** -19 * raw.abs().amax()).all()
    assert torch.equal(c.rows(1, slots), v0) and torch.equal(v.double(), v0)


def test_append_rows_that_8_bits_cannot_hold():
    """Zeros and the smallest rows become 0, a row with an infinity or a NaN becomes NaN, the next row is unaffected."""
    g = gen(4)
    x = normal(g, 6, 1, 64)
    x[1] = 0
    x[2] *= 1e-36
    x[3, 0, 5] = math.inf
    x[4, 0, 63] = math.nan
    c = Cache(g, S8, 1, 8, 1, 64, False)
    out = torch.empty(6, 1, 64, dtype=BF16, device="cuda")
    api.pulpnn_kv_append(c.handle, torch.arange(6, device="cuda"), x, x, k_out=out)
    torch.cuda.synchronize()
    got = c.rows(0, torch.arange(6, device="cuda"))
    assert (got[1] == 0).all() and (got[2] == 0).all()
    assert got[3].isnan().all() and got[4].isnan().all()
    for i in (0, 5):
        assert ((got[i] - x[i].double()).abs() <= x[i].abs().max().double() / 127 * 0.51).all()
    assert torch.equal(out, x.to(BF16)) or (out.isnan() == x.isnan()).all()


@pytest.mark.parametrize("cache,wide", [(S8, BF16), (S8, F16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("n,hkv,dim,heads_first,page", [(1, 1, 16, False, 1), (75, 3, 80, True, 20), (333, 8, 128, False, 16), (50, 2, 64, True, 7)])
def test_gather(cache, wide, n, hkv, dim, heads_first, page):
    g = gen(n)
    c = Cache(g, cache, 5, page, hkv, dim, heads_first)
    slots = torch.randint(0, 5 * page, (n,), generator=g, device="cuda")       # the same slot more than once, too
    bad = torch.zeros(n, dtype=torch.bool, device="cuda")
    if n > 9:
        slots[3], slots[7], slots[9] = -1, 5 * page, -2 ** 62
        bad[[3, 7, 9]] = True
    k, v = Fenced((n, hkv, dim), wide), Fenced((n, hkv, dim), wide)
    api.pulpnn_kv_gather(c.handle, slots, k.view, v.view)
    only = Fenced((n, hkv, dim), wide)
    api.pulpnn_kv_gather(c.handle, slots, None, only.view)
    torch.cuda.synchronize()
    assert k.intact() and v.intact() and only.intact() and c.intact()
    for i, x in enumerate((k, v)):
        want = c.rows(i, slots.where(~bad, torch.zeros_like(slots)))
        want[bad] = 0
        # a product in 32 bits, rounded to 16
        assert ((x.view.double() - want).abs() <= (eps(wide) / 2 + 2.0 ** -23) * want.abs()).all()
    assert torch.equal(only.view, v.view)


# ---- one token per sequence -----------------------------------------------------------------------------

def decode_case(seed, lens, hq, hkv, dim, q_type, cache_type, page, heads_first, window=0, u8=False, extra_pages=0, bad=False, big=1.0):
    g = gen(seed)
    pages_of = [-(-n // page) for n in lens]
    width = max(pages_of + [1]) + extra_pages
    total = sum(pages_of) + 2
    c = Cache(g, cache_type, total, page, hkv, dim, heads_first)
    order = torch.randperm(total, generator=g, device="cuda")
    table = torch.full((len(lens), width), -7, dtype=torch.int32, device="cuda")      # entries that must not be used
    at = 0
    for b, n in enumerate(pages_of):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    if bad:
        for b, n in enumerate(pages_of):
            if n > 1:
                table[b, n // 2] = (-1, total, 2 ** 31 - 1)[b % 3]
    # the rows behind each sequence's last one, and the pages nobody has, hold NaN
    if cache_type != S8:
        for x in (c.k, c.v):
            y = x.view.transpose(1, 2) if heads_first else x.view
            y[order[at:]] = math.nan
            for b, n in enumerate(lens):
                if n % page:
                    y[table[b, n // page].long(), n % page:] = math.nan
    q = Fenced((len(lens), hq, dim), q_type, fill=normal(g, len(lens), hq, dim) * big)
    out = Fenced((len(lens), hq, dim), torch.uint8 if u8 else q_type)
    lse = torch.full((len(lens), hq), 7.0, device="cuda")
    n_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    scale = dim ** -0.5
    step = 0.02 if u8 else None
    api.pulpnn_attn_decode(c.handle, q.view, table, n_t, out.view, window=window, lse=lse, out_step=step, out_zero=128 if u8 else 0)
    torch.cuda.synchronize()
    assert out.intact() and c.intact()
    group = hq // hkv
    for b, n in enumerate(lens):
        t = torch.arange(max(0, n - window) if window else 0, n, device="cuda")
        page_of = table[b].long()[t // page]
        fine = (page_of >= 0) & (page_of < total)
        slots = (page_of * page + t % page)[fine]
        k, v = c.rows(0, slots), c.rows(1, slots)
        for h in range(hq):
            m = len(slots)
            want, want_lse, weighted, product = attend(q.view[b, h:h + 1].double(), k[:, h // group], v[:, h // group],
                                                       torch.ones(1, m, dtype=torch.bool, device="cuda"), scale)
            if m == 0:
                assert lse[b, h] == -math.inf
                assert (out.view[b, h] == (128 if u8 else 0)).all()
                continue
            # an 8-bit cache's weights are multiplied in fp16, and q in fp16 with 24 bits below its largest value
            weight = F16 if cache_type == S8 else q_type
            tol = tolerance(want, weighted, product, m, dim, None if u8 else q_type, weight)
            if u8:
                got = out.view[b, h].double()
                exact = (want[0] / step + 128).clamp(0, 255)
                assert ((got - exact).abs() <= 0.5 + tol[0] / step + 1e-4).all()
            else:
                assert ((out.view[b, h].double() - want[0]).abs() <= tol[0]).all(), (b, n, h)
            assert abs(lse[b, h].double() - want_lse) <= lse_tolerance(want_lse, product, m, dim)


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 257, 500]


@pytest.mark.parametrize("q_type,cache", [(BF16, BF16), (F16, F16), (BF16, S8), (F16, S8)])
@pytest.mark.parametrize("hq,hkv,dim,page,heads_first", [(8, 2, 128, 16, False), (3, 3, 80, 20, True), (7, 1, 64, 1, False), (12, 1, 112, 7, True),
                                                        (40, 2, 128, 64, True), (2, 1, 16, 33, False), (16, 2, 96, 16, False)])
def test_decode(q_type, cache, hq, hkv, dim, page, heads_first):
    decode_case(dim + hq, LENS, hq, hkv, dim, q_type, cache, page, heads_first)


@pytest.mark.parametrize("dim", [72, 80, 88])
@pytest.mark.parametrize("hq,hkv,page,heads_first,window", [(4, 4, 16, False, 0), (10, 1, 32, True, 0), (6, 2, 48, False, 77), (20, 2, 20, False, 0),
                                                            (2, 2, 9, True, 130)])
def test_decode_rows_as_long_as_they_are(dim, hq, hkv, page, heads_first, window):
    """65 to 80 channels lie in shared memory without gaps, more in boxes of 64."""
    decode_case(dim * 3 + hq, LENS, hq, hkv, dim, F16, F16, page, heads_first, window=window, extra_pages=1)


@pytest.mark.parametrize("cache", [BF16, S8])
@pytest.mark.parametrize("window", [1, 16, 100, 10 ** 9])
def test_decode_window(cache, window):
    decode_case(5, LENS, 4, 2, 64, BF16, cache, 20, False, window=window)


@pytest.mark.parametrize("cache,lens", [(F16, [5000, 3, 12345]), (S8, [9001, 0, 20000]), (BF16, [70000])])
def test_decode_long(cache, lens):
    decode_case(6, lens, 8, 2, 128, F16 if cache == F16 else BF16, cache, 64, False)


@pytest.mark.parametrize("cache", [F16, S8])
def test_decode_uint8_output(cache):
    decode_case(7, [1, 40, 300], 4, 2, 128, F16, cache, 16, False, u8=True)


@pytest.fixture
def forced_split():
    yield lambda n: api.set_option(api.OPT_SPLIT_K, n)
    api.set_option(api.OPT_SPLIT_K, 0)


@pytest.mark.parametrize("cache,page,dim", [(BF16, 16, 128), (S8, 32, 64), (S8, 20, 128), (F16, 7, 80)])
@pytest.mark.parametrize("split", [1, 2, 3, 7, 8, 16, 40, 600])
def test_decode_splits(forced_split, split, cache, page, dim):
    """However many CTAs and clusters share a sequence (600: more than there are tiles), empty sequences among them."""
    forced_split(split)
    decode_case(split, [0, 1, 130, 1000, 33], 12, 1, dim, F16 if cache == F16 else BF16, cache, page, False)
    if split >= 16:
        assert api.last_kernel() == "attn_join_kernel"


def test_decode_splits_uint8_output(forced_split):
    forced_split(24)
    decode_case(7, [1, 40, 0, 700], 4, 2, 72, F16, F16, 16, False, u8=True)


def test_decode_one_long_sequence_is_shared_by_clusters():
    decode_case(13, [60000], 4, 1, 128, BF16, BF16, 16, False)
    assert api.last_kernel() == "attn_join_kernel"


def test_decode_captured_and_on_several_streams_at_once():
    """Calls that need memory for their parts: captured into two graphs that are replayed side by side with a third, eager
    stream, lengths changing between replays."""
    g = gen(14)
    dim, page, pages = 128, 16, 2048
    c = Cache(g, BF16, 2 * pages, page, 1, dim, False)
    tables = [torch.randperm(2 * pages, generator=g, device="cuda")[:pages].to(torch.int32)[None].contiguous() for _ in range(3)]
    q = [normal(g, 1, 4, dim, dtype=BF16) for _ in range(3)]
    lens = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(3)]
    out, want = [torch.empty_like(x) for x in q], []
    streams = [torch.cuda.Stream() for _ in range(3)]
    graphs = []
    torch.cuda.synchronize()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        api.set_stream(streams[i])
        with torch.cuda.graph(graph, stream=streams[i]):
            api.pulpnn_attn_decode(c.handle, q[i], tables[i], lens[i], out[i])
        assert api.last_kernel() == "attn_join_kernel"
        graphs.append(graph)
    for turn, n in enumerate((30000, 17, 0, 32768)):
        for i in range(3):
            lens[i].fill_(max(0, n - 100 * i))
        torch.cuda.synchronize()
        for _ in range(3):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
            api.set_stream(streams[2])
            api.pulpnn_attn_decode(c.handle, q[2], tables[2], lens[2], out[2])
        api.set_stream(None)
        torch.cuda.synchronize()
        for i in range(3):
            m = max(0, n - 100 * i)
            t = torch.arange(m, device="cuda")
            slots = tables[i][0].long()[t // page] * page + t % page
            k, v = (c.rows(w, slots)[:, 0] for w in range(2))
            want, _, sums, product = attend(q[i][0].double(), k, v, torch.ones(4, m, dtype=torch.bool, device="cuda"), dim ** -0.5)
            if m == 0:
                assert (out[i] == 0).all()
            else:
                assert ((out[i][0].double() - want).abs() <= tolerance(want, sums, product, m, dim, BF16, BF16)).all(), (turn, i)


def test_calls_of_several_threads():
    """Each host thread has a context, a stream and its own results."""
    import threading
    g = gen(15)
    c = Cache(g, S8, 600, 16, 2, 64, False)
    jobs, errors = [], []
    for i in range(4):
        n = 2000 * i + 150
        q = normal(g, 1, 8, 64, dtype=BF16)
        table = torch.randperm(600, generator=g, device="cuda")[:(n + 15) // 16].to(torch.int32)[None].contiguous()
        lens = torch.tensor([n], dtype=torch.int32, device="cuda")
        want = torch.empty_like(q)
        api.pulpnn_attn_decode(c.handle, q, table, lens, want)
        p = normal(g, 200 + i, 4, 64, dtype=F16)
        cu = torch.tensor([0, 200 + i], dtype=torch.int32, device="cuda")
        pw = torch.empty_like(p)
        api.pulpnn_attn_prompt(p, p[:, :2], p[:, 2:], cu, pw)
        jobs.append((q, table, lens, want, p, cu, pw))
    torch.cuda.synchronize()

    def work(i):
        try:
            api.set_device(0)
            stream = torch.cuda.Stream()
            api.set_stream(stream)
            q, table, lens, want, p, cu, pw = jobs[i]
            for _ in range(20):
                out, po = torch.empty_like(q), torch.empty_like(p)
                stream.wait_stream(torch.cuda.current_stream())
                api.pulpnn_attn_decode(c.handle, q, table, lens, out)
                api.pulpnn_attn_prompt(p, p[:, :2], p[:, 2:], cu, po)
                api.synchronize()
                assert torch.equal(out, want) and torch.equal(po, pw)
            assert api.device_status() == 0
        except BaseException as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize("cache", [BF16, S8])
def test_decode_pages_outside_the_cache_are_left_out(cache):
    decode_case(8, [40, 100, 700, 33], 4, 1, 64, BF16, cache, 16, False, bad=True, extra_pages=3)


@pytest.mark.parametrize("cache", [F16, S8])
def test_decode_large_scores(cache):
    """Scores of several hundred: the running maximum is raised many times, and most weights vanish."""
    decode_case(9, [1, 77, 900], 4, 2, 128, F16, cache, 16, True, big=60.0)


def test_decode_scales_that_differ_by_powers_of_ten():
    """Rows of an 8-bit cache whose scales span 2^60: each row's weight keeps fp16's precision."""
    g = gen(10)
    c = Cache(g, S8, 8, 16, 1, 64, False)
    c.s[1].view.copy_(2.0 ** (torch.rand(8, 16, 1, generator=g, device="cuda") * 60 - 40))
    c.s[0].view.copy_(torch.full((8, 16, 1), 0.01))
    q = normal(g, 1, 2, 64, dtype=BF16)
    out = torch.empty_like(q)
    api.pulpnn_attn_decode(c.handle, q, torch.arange(8, device="cuda", dtype=torch.int32)[None], torch.tensor([128], device="cuda", dtype=torch.int32), out)
    torch.cuda.synchronize()
    k, v = (c.rows(i, torch.arange(128, device="cuda"))[:, 0] for i in range(2))
    want, _, weighted, product = attend(q[0].double(), k, v, torch.ones(2, 128, dtype=torch.bool, device="cuda"), 64 ** -0.5)
    assert ((out[0].double() - want).abs() <= tolerance(want, weighted, product, 128, 64, BF16, F16)).all()


def test_decode_lengths_beyond_the_table_are_cut():
    g = gen(11)
    c = Cache(g, BF16, 3, 16, 1, 64, False)
    q = normal(g, 2, 1, 64, dtype=BF16)
    table = torch.tensor([[0, 1], [2, 0]], device="cuda", dtype=torch.int32)
    outs = []
    for lens in ((32, 0), (2 ** 31 - 1, -5)):
        out = torch.empty_like(q)
        api.pulpnn_attn_decode(c.handle, q, table, torch.tensor(lens, device="cuda", dtype=torch.int32), out)
        outs.append(out)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and (outs[1][1] == 0).all()


def test_decode_is_the_same_every_time_and_beyond_32_bit_offsets():
    """A cache of 2^32 elements and more: its last pages. Twice the same call gives the same bits."""
    pages, page, hkv, dim = 2100000, 16, 1, 128
    k = torch.empty((pages, page, hkv, dim), dtype=S8, device="cuda")
    v = torch.empty_like(k)
    s = torch.full((pages, page, hkv), 0.01, device="cuda")
    g = gen(12)
    for x in (k, v):
        x[:8].copy_(torch.randint(-127, 128, (8, page, hkv, dim), generator=g, device="cuda"))
        x[-8:].copy_(torch.randint(-127, 128, (8, page, hkv, dim), generator=g, device="cuda"))
    cache = api.KVCache(k, v, s, s.clone())
    q = normal(g, 1, 4, dim, dtype=BF16)
    table = torch.cat([torch.arange(pages - 8, pages), torch.arange(8)]).to(torch.int32).cuda()[None]
    n = torch.tensor([250], dtype=torch.int32, device="cuda")
    outs = []
    for _ in range(2):
        out = torch.empty_like(q)
        api.pulpnn_attn_decode(cache, q, table, n, out)
        outs.append(out)
    slots = (table[0].long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[:250]
    rows = [x.view(-1, dim)[slots].double() * 0.01 for x in (k, v)]
    want, _, weighted, product = attend(q[0].double(), rows[0], rows[1], torch.ones(4, 250, dtype=torch.bool, device="cuda"), dim ** -0.5)
    tol = tolerance(want, weighted, product, 250, dim, BF16, F16) + 1e-6 * weighted[0]       # the scale 0.01 in 32 bits
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1])
    assert ((outs[0][0].double() - want).abs() <= tol).all()
    # and rows stored there, and read back
    x = normal(g, 3, 1, dim, dtype=BF16)
    at = torch.tensor([pages * page - 1, pages * page - 40, 5], device="cuda")
    back = torch.empty_like(x)
    api.pulpnn_kv_append(cache, at, x, x)
    api.pulpnn_kv_gather(cache, at, back)
    torch.cuda.synchronize()
    assert ((back.double() - x.double()).abs() <= x.double().abs().amax(-1, keepdim=True) * (0.51 / 127 + 2.0 ** -8)).all()


# ---- whole prompts ------------------------------------------------------------------------------------------

def prompt_case(seed, lens, before, hq, hkv, dim, dtype, causal=True, window=0, pad=0, u8=False, poison=False, big=1.0, packed=False):
    """before[b]: keys ahead of the first query (negative: fewer keys than queries)."""
    g = gen(seed)
    nk_of = [a + b for a, b in zip(lens, before)]
    nq, nk = sum(lens) + pad, sum(nk_of) + pad
    if packed:
        whole = normal(g, nq, hq + 2 * hkv, dim, dtype=dtype)
        q, k, v = whole[:, :hq], whole[:, hq:hq + hkv], whole[:, hq + hkv:]
        q.mul_(big)
    else:
        q, k, v = (Fenced((n, h, dim), dtype, fill=normal(g, n, h, dim) * f).view for n, h, f in ((nq, hq, big), (nk, hkv, 1), (nk, hkv, 1)))
    if poison:
        for t in (k, v):       # what no query of its own sequence sees, or only later ones do
            t[nk - pad:] = math.nan
            at = 0
            for a, n in zip(lens, nk_of):
                if n > 3 and a > 2:
                    t[at + n - 1] = math.inf
                    t[at + n - 2, :, ::3] = math.nan if t is v else -math.inf
                at += n
    out = Fenced((nq, hq, dim), torch.uint8 if u8 else dtype)
    out.view.fill_(3)
    lse = torch.full((nq, hq), 9.0, device="cuda")
    cu_q = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    cu_k = torch.tensor([0] + nk_of, device="cuda").cumsum(0).to(torch.int32)
    step = 0.02 if u8 else None
    api.pulpnn_attn_prompt(q, k, v, cu_q, out.view, cu_k=cu_k, causal=causal, window=window, lse=lse, out_step=step, out_zero=100 if u8 else 0)
    torch.cuda.synchronize()
    assert api.last_kernel() == "attn_prompt_kernel"
    assert api.device_status() == 0
    assert out.intact()
    q0 = k0 = 0
    scale, group = dim ** -0.5, hq // hkv
    for a, b in zip(lens, before):
        n = a + b
        pos = torch.arange(a, device="cuda")[:, None] + b
        j = torch.arange(n, device="cuda")
        seen = (j <= pos) if causal else torch.ones(a, n, dtype=torch.bool, device="cuda")
        if window:
            seen = seen & (j > pos - window)
        for h in range(hq):
            kk, vv = (t[k0:k0 + n, h // group].double() for t in (k, v))
            got, got_lse = out.view[q0:q0 + a, h].double(), lse[q0:q0 + a, h].double()
            qq = q[q0:q0 + a, h].double()
            if poison:
                # rows that see nothing that is not a number; for the others only that they say so
                odd_k, odd_v = ~kk.isfinite().all(1), ~vv.isfinite()
                clean = ~(seen & (odd_k | odd_v.any(1))).any(1)
                kk, vv = kk.where(~odd_k[:, None], torch.zeros_like(kk)), vv.where(~odd_v, torch.zeros_like(vv))
                assert (~got[~clean].isfinite()).any(1).all()
                assert got[clean].isfinite().all()
                seen_h, rows = seen & ~(odd_k | odd_v.any(1)), clean
            else:
                seen_h, rows = seen, torch.ones(a, dtype=torch.bool, device="cuda")
            want, want_lse, weighted, product = attend(qq, kk, vv, seen_h, scale)
            none = ~seen_h.any(1)
            assert (got[none & rows] == (100 if u8 else 0)).all() and (got_lse[none & rows] == -math.inf).all()
            rows = rows & ~none
            tol = tolerance(want, weighted, product, n, dim, None if u8 else dtype, dtype)
            if u8:
                exact = (want / step + 100).clamp(0, 255)
                assert ((got - exact).abs() <= 0.5 + tol / step + 1e-4)[rows].all()
            else:
                assert ((got - want).abs() <= tol)[rows].all(), (a, b, h, ((got - want).abs() / tol)[rows].max())
            assert ((got_lse - want_lse).abs() <= lse_tolerance(want_lse, product, n, dim))[rows].all()
        q0, k0 = q0 + a, k0 + n
    assert (out.view[q0:] == 3).all() and (lse[q0:] == 9).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,hkv,dim", [(4, 1, 128), (2, 2, 64), (3, 1, 80), (7, 1, 112), (1, 1, 8), (2, 1, 72)])
def test_prompt_smallest(dtype, hq, hkv, dim):
    prompt_case(1, [1, 5], [0, 0], hq, hkv, dim, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,hkv,dim", [(4, 1, 128), (2, 2, 64), (3, 1, 80), (7, 1, 112), (2, 2, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt(dtype, hq, hkv, dim, causal):
    prompt_case(2, [0, 127, 128, 0, 129, 1, 256, 300, 77], [0] * 9, hq, hkv, dim, dtype, causal=causal, pad=11)


@pytest.mark.parametrize("causal", [True, False])
def test_prompt_with_a_cached_beginning(causal):
    """More keys than queries, none at all, and fewer: then the first queries see nothing."""
    prompt_case(3, [5, 130, 1, 200, 40, 300], [300, 1, 511, -150, -40, -1], 4, 2, 128, BF16, causal=causal, pad=3)


@pytest.mark.parametrize("window", [1, 64, 128, 200, 2 ** 31 - 1])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (4, 1)])
def test_prompt_window(window, hq, hkv):
    prompt_case(4, [700, 130, 3], [0, 300, 200], hq, hkv, 64, F16, window=window)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
def test_prompt_what_is_masked_does_not_reach_the_result(dtype, dim):
    prompt_case(5, [130, 5, 300, 128], [0, 20, 0, 0], 2, 1, dim, dtype, poison=True, pad=40)


def test_prompt_uint8_output_and_packed_inputs():
    prompt_case(6, [200, 61], [0, 0], 4, 2, 128, BF16, u8=True)
    prompt_case(6, [200, 61], [0, 0], 4, 2, 80, F16, packed=True)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prompt_large_scores(dtype):
    """Scores of several hundred: the reference is raised in many tiles, and the sums rescaled."""
    prompt_case(7, [900], [0], 2, 1, 128, dtype, big=60.0, causal=False)


@pytest.mark.parametrize("dtype,dim,n", [(BF16, 128, 5000), (F16, 64, 3333)])
def test_prompt_long(dtype, dim, n):
    prompt_case(8, [n], [0], 2, 1, dim, dtype)


def test_prompt_many_sequences():
    """More sequences than a CTA has threads, most of them empty or of a few rows."""
    lens = [(i * 37) % 5 if i % 50 else 140 for i in range(1000)]
    prompt_case(9, lens, [0] * 1000, 1, 1, 64, BF16)


@pytest.mark.parametrize("seqs", [2, 33, 180, 256, 257])
@pytest.mark.parametrize("hq,hkv", [(14, 2), (8, 8)])
def test_prompt_sequences_taken_longest_first_or_in_order(seqs, hq, hkv):
    lens = [(b * 37) % 61 if b % 3 else (b * 131) % 400 for b in range(seqs)]
    lens[-1] = 390
    prompt_case(seqs, lens, [0] * seqs, hq, hkv, 64, BF16, pad=2)


def test_prompt_offsets_that_make_no_sense_stay_inside():
    g = gen(20)
    q, k, v = (normal(g, 200, 1, 64, dtype=BF16) for _ in range(3))
    out = Fenced((200, 1, 64), BF16)
    cu = torch.tensor([-5, 2 ** 31 - 1, 100, 50, 400, -2 ** 31, 150], dtype=torch.int32, device="cuda")
    api.pulpnn_attn_prompt(q, k, v, cu, out.view)
    api.pulpnn_attn_prompt(q, k, v, cu, out.view, cu_k=cu.flip(0).contiguous())
    torch.cuda.synchronize()
    assert out.intact() and api.device_status() == 0


# ---- as they are used ---------------------------------------------------------------------------------------

def test_a_decoder_layers_attention_between_8_bit_fully_connected_layers():
    """The projection's accumulators are rotated and stored, a prompt is attended to, tokens follow one by one, and the uint8
    result feeds the next fully connected layer: in a stream of its own, the token steps as a captured graph."""
    rng = np.random.default_rng(5)
    hq, hkv, dim, page, n0, steps = 4, 2, 64, 16, 150, 20
    hidden, total = 256, n0 + steps
    w_np = rng.integers(-20, 20, size=((hq + 2 * hkv) * dim, hidden)).astype(np.int8)
    w2_np = rng.integers(-20, 20, size=(hidden, hq * dim)).astype(np.int8)
    x_np = rng.integers(0, 256, size=(total, hidden), dtype=np.uint8)
    w, w2, x = (torch.from_numpy(t).cuda() for t in (w_np, w2_np, x_np))
    rows = (hq + 2 * hkv) * dim
    step = torch.from_numpy(rng.uniform(0.5, 1.5, size=rows).astype(np.float32) * 2e-5).cuda()
    sq, sk, sv = step[:hq * dim].clone(), step[hq * dim:(hq + hkv) * dim].clone(), step[(hq + hkv) * dim:].clone()
    freq = freqs(dim)
    pages = -(-total // page)
    order = torch.randperm(pages + 3, generator=gen(1), device="cuda")[:pages]
    table = order.to(torch.int32)[None].contiguous()
    t = torch.arange(total, device="cuda")
    all_slots = order[t // page] * page + t % page
    kc, vc = (torch.zeros(pages + 3, page, hkv, dim, dtype=S8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(pages + 3, page, hkv, device="cuda") for _ in range(2))
    cache = api.KVCache(kc, vc, ks, vs)

    def project(src, dst, n):
        api.set_batch(n)
        api.pulp_nn_linear_out_32(32, src, None, dst, w, hidden, rows)
        api.set_batch(1)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    api.set_stream(stream)
    try:
        with torch.cuda.stream(stream):
            acc = torch.empty(n0, hq + 2 * hkv, dim, dtype=S32, device="cuda")
            q, k, v = (torch.empty(n0, h, dim, dtype=BF16, device="cuda") for h in (hq, hkv, hkv))
            o = torch.empty(n0, hq, dim, dtype=BF16, device="cuda")
            cu = torch.tensor([0, n0], dtype=torch.int32, device="cuda")
            project(x[:n0].contiguous(), acc, n0)
            api.pulpnn_kv_append(cache, all_slots[:n0], acc[:, hq:hq + hkv], acc[:, hq + hkv:], positions=t[:n0].to(torch.int32), inv_freq=freq,
                                 q=acc[:, :hq], q_out=q, k_out=k, v_out=v, q_step=sq, k_step=sk, v_step=sv)
            api.pulpnn_attn_prompt(q, k, v, cu, o)
            # buffers of a token step
            x1 = torch.empty(1, hidden, dtype=torch.uint8, device="cuda")
            acc1 = torch.empty(1, hq + 2 * hkv, dim, dtype=S32, device="cuda")
            q1 = torch.empty(1, hq, dim, dtype=BF16, device="cuda")
            pos1 = torch.zeros(1, dtype=torch.int32, device="cuda")
            slot1 = torch.zeros(1, dtype=torch.int64, device="cuda")
            len1 = torch.zeros(1, dtype=torch.int32, device="cuda")
            o1 = torch.empty(1, hq, dim, dtype=torch.uint8, device="cuda")
            y1 = torch.empty(1, hidden, dtype=S32, device="cuda")

            def token():
                project(x1, acc1, 1)
                api.pulpnn_kv_append(cache, slot1, acc1[:, hq:hq + hkv], acc1[:, hq + hkv:], positions=pos1, inv_freq=freq, q=acc1[:, :hq],
                                     q_out=q1, q_step=sq, k_step=sk, v_step=sv)
                api.pulpnn_attn_decode(cache, q1, table, len1, o1, out_step=0.05, out_zero=128)
                api.pulp_nn_linear_out_32(32, o1, None, y1, w2, hq * dim, hidden)

            def load(i):
                x1.copy_(x[i:i + 1])
                pos1.fill_(i)
                slot1.copy_(all_slots[i:i + 1])
                len1.fill_(i + 1)

            load(n0)
            token()                                        # once outside the graph
            first = (o1.clone(), y1.clone())
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                token()
            got = []
            for i in range(n0, total):
                load(i)
                graph.replay()
                got.append((o1.clone(), y1.clone()))
        torch.cuda.synchronize()
    finally:
        api.set_stream(None)
    assert torch.equal(first[0], got[0][0]) and torch.equal(first[1], got[0][1])

    # the definition, in 64 bits, from the same bytes
    acc_all = (x.double() @ w.double().T).view(total, hq + 2 * hkv, dim) * step.double().view(1, -1, dim)
    qq, kk = (rotate(a, t, freq, False) for a in (acc_all[:, :hq], acc_all[:, hq:hq + hkv]))
    vv = acc_all[:, hq + hkv:]
    seen = t[:n0, None] >= t[None, :n0]
    for h in range(hq):
        want, _, weighted, product = attend(qq[:n0, h], kk[:n0, h // 2], vv[:n0, h // 2], seen, dim ** -0.5)
        # q, k and v were rounded to bf16: each score moves by 2 x 2^-8 of the sum of |q||k|, v by 2^-8
        tol = tolerance(want, weighted, product, n0, dim, BF16, BF16) + (2.0 ** -8 + 2 * 2.1 * 2.0 ** -8 * product[:, None]) * weighted[0]
        assert ((o[:, h].double() - want).abs() <= tol).all()
    for i in range(n0, total):
        o_got, y_got = got[i - n0]
        rows_k, rows_v = (c_[all_slots[:i + 1] // page, all_slots[:i + 1] % page].double() * s_[all_slots[:i + 1] // page, all_slots[:i + 1] % page].double()[..., None]
                          for c_, s_ in ((kc, ks), (vc, vs)))
        for r, full in ((rows_k, kk[:i + 1]), (rows_v, vv[:i + 1])):
            most = full.abs().amax(-1, keepdim=True)
            assert ((r - full).abs() <= most * (0.5 / 127 + 1e-5)).all()
        for h in range(hq):
            want, _, weighted, product = attend(qq[i:i + 1, h], rows_k[:, h // 2], rows_v[:, h // 2], torch.ones(1, i + 1, dtype=torch.bool, device="cuda"), dim ** -0.5)
            tol = tolerance(want, weighted, product, i + 1, dim, None, F16) + 2.1 * 2.0 ** -8 * product[:, None] * weighted[0]
            exact = (want / 0.05 + 128).clamp(0, 255)
            assert ((o_got[0, h].double() - exact).abs() <= 0.5 + tol / 0.05 + 1e-4).all()
        want_y = (o_got.view(1, -1).double() @ w2.double().T).to(torch.int64)
        assert torch.equal(y_got.to(torch.int64), want_y)
