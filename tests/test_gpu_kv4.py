"""The paged 4-bit cache and the attention over it against 64-bit arithmetic.

Written codes and scales: equal to the definition (quotients exact in 64 bits
at every tie a 16-bit input can meet). Read values: one rounding to the type.

Attention: with Q and the cache exact, a score's error is that of its f32
accumulation, at most (Dh / 16 + 6) roundings of 2^-23 of the sum of |q k| --
call it ds --, each weight is off by a factor within 2 ds, the exponential's
2^-21 and, for the 16-bit types, the 2^-11 of an f16 weight (f32 queries
split it: 2^-21); the weighted sums add one 2^-23 per 16 keys of a warp's run
and per joined part. So |O - exact| <= (2 ds + w + n 2^-23) sum_t p_t |v_t|,
plus half a step of the output's type. Below the normal f16 range a weight is off
by half a subnormal step instead: the kernels hold exp(s - max) in f16 times 2^15
(long prompt chunks: the largest one between 2^7 and 2^15), whose subnormal step
is 2^-24, so a weight relative to the largest one is off by at most 2^-25 / 2^15 =
2^-40 (chunks: 2^-32), and O (divided by a sum of at least 1) by as much of
sum_t |v_t|. (It shows where the heavy keys hold zeros in a column.) The
output's half step is eps / 2 of the value, or half the subnormal step, which is
smallest_normal * eps / 2, for values that f16 holds as subnormals."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

E2M1 = [0, 0.5, 1, 1.5, 2, 3, 4, 6]


def _dt(t):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[t]


def _half_step(v, dtype):
    import torch
    f = torch.finfo(dtype)
    return v.clamp(min=f.smallest_normal) * f.eps / 2


def _lut():
    import torch
    return torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device="cuda")


def _decode(codes, scales, gs):
    """[pages][Hkv][page][Dh] in 64 bits."""
    import torch
    c = codes.long()
    v = torch.stack((c & 15, c >> 4), -1).flatten(-2)
    s = scales.view(torch.float8_e4m3fn).double().repeat_interleave(16, -1)
    return _lut()[v] * s * gs.double()[None, :, None, None]


def _quantize(x, g):
    """Codes and e4m3 scales of x [..., Dh] by the definition; g broadcast over blocks."""
    import torch
    b = x.double().unflatten(-1, (-1, 16))
    m = b.abs().nan_to_num(0, posinf=math.inf).amax(-1)
    s = (m.float() / (6 * g)).clamp(max=448).to(torch.float8_e4m3fn)
    step = (s.double() * g.double())[..., None]
    z = torch.where(step > 0, b / step, torch.zeros_like(b))
    grid = _lut()[:8]
    mid = (grid[1:] + grid[:-1]) / 2
    k = torch.bucketize(z.abs(), mid)
    k = torch.where((k < 7) & (k % 2 == 1) & (z.abs() == mid[k.clamp(max=6)]), k + 1, k)
    k = torch.where(z.isnan(), torch.full_like(k, 7), k + 8 * ((z < 0) & (k > 0)))
    k = k.flatten(-2)
    return (k[..., 0::2] | (k[..., 1::2] << 4)).to(torch.uint8), s.view(torch.uint8)


def _cache(rb, pages, Hkv, page, Dh, seed, gs=True):
    """A cache of random codes, its scales between 2^-3 and 2; slots nothing wrote are poisoned by the tests."""
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    by = lambda n: torch.randint(0, 256, (pages, Hkv, page, n), generator=g, device="cuda").to(torch.uint8)  # noqa: E731
    sc = lambda: torch.randint(32, 65, (pages, Hkv, page, Dh // 16), generator=g, device="cuda").to(torch.uint8)  # noqa: E731
    gg = lambda: (0.3 + torch.rand(Hkv, generator=g, device="cuda")) if gs else None  # noqa: E731
    return rb.KV4Cache(by(Dh // 2), sc(), by(Dh // 2), sc(), gg(), gg())


def _reference(cache, q, lens, table, nqs, causal, window, scale, tiny_step=2.0 ** -40):
    """O and the tolerance's parts in 64 bits, sequence by sequence."""
    import torch
    kc, ks, vc, vs, gk, gv = cache.tensors
    one = torch.ones(cache.Hkv, device="cuda")
    K, V = _decode(kc, ks, gk if gk is not None else one), _decode(vc, vs, gv if gv is not None else one)
    Hq = q.shape[1]
    G = Hq // cache.Hkv
    out, spread, ds, tiny = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(4))
    at = 0
    for b, (n, nq) in enumerate(zip(lens, nqs)):
        for i in range(nq):
            p = n - nq + i
            hi = max(0, min(n, p + 1)) if causal else n
            lo = max(0, p - window + 1) if window else 0
            if hi > lo:
                t = torch.arange(lo, hi, device="cuda")
                pg, off = table[b].long()[t // cache.page], t % cache.page
                k = K[pg, :, off].repeat_interleave(G, 1)
                v = V[pg, :, off].repeat_interleave(G, 1)
                z = torch.einsum("hd,thd->ht", q[at].double(), k) * scale
                za = torch.einsum("hd,thd->ht", q[at].double().abs(), k.abs()) * scale
                w = torch.softmax(z, 1)
                out[at] = torch.einsum("ht,thd->hd", w, v)
                spread[at] = torch.einsum("ht,thd->hd", w, v.abs())
                tiny[at] = tiny_step * v.abs().sum(0)
                ds[at] = (za.amax(1) * (cache.Dh / 16 + 6) * 2.0 ** -23)[:, None]
            at += 1
    return out, spread, ds, tiny


def _attend(rb, cache, t, lens, nqs, Hq, causal=1, window=0, scale=0.0, seed=0, extra=0, table=None):
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    per = max(1, max(-(-n // cache.page) for n in lens))
    if table is None:
        order = torch.randperm(cache.pages, generator=g, device="cuda").int()
        table = torch.full((len(lens), per), 1 << 30, dtype=torch.int32, device="cuda")  # (never read past a length)
        at = 0
        for b, n in enumerate(lens):
            k = -(-n // cache.page)
            table[b, :k] = order[at:at + k]
            at += k
    T = sum(nqs)
    q = torch.randn(T + extra, Hq, cache.Dh, generator=g, device="cuda").to(_dt(t))
    O = torch.full_like(q, 77.0)
    lens_d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu = torch.tensor(np.concatenate(([0], np.cumsum(nqs))), dtype=torch.int32, device="cuda")
    single = all(n == 1 for n in nqs)
    rb.attention_kv4(q, cache, lens_d, table, cu_q=None if single else cu, max_q=1 if single else max(max(nqs), 1),
                     O=O, scale=scale, causal=causal, window=window)
    return q, O, table, lens_d, cu


def _check(rb, cache, t, lens, nqs, Hq, causal=1, window=0, scale=0.0, tiny_step=2.0 ** -40, **kw):
    import torch
    q, O, table, _, _ = _attend(rb, cache, t, lens, nqs, Hq, causal, window, scale, **kw)
    rb.sync_status()
    T = sum(nqs)
    want, spread, ds, tiny = _reference(cache, q, lens, table, nqs, causal, window, scale or 1 / math.sqrt(cache.Dh),
                                        tiny_step)
    w = 2.0 ** -21 + (2.0 ** -21 if t == "f32" else 2.0 ** -11)
    n = max(max(lens), 16) / 16 + 64
    tol = (2 * ds + w + n * 2.0 ** -23) * spread + tiny
    tol = tol + _half_step(want.abs() + tol, q.dtype)
    d = (O[:T].double() - want[:T]).abs()
    assert (d <= tol[:T]).all(), ((d / tol[:T].clamp(min=1e-300)).nan_to_num(math.inf).max().item(), d.max().item())
    assert (O[T:] == 77).all()
    return O


# ------------------------------------------------------------------ write, read

@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,Hkv,Dh,page,gs", [(1, 1, 16, 16, False), (5, 2, 64, 16, True), (70, 3, 80, 48, True),
                                              (300, 8, 128, 64, True), (33, 1, 256, 32, False)])
def test_write_and_read(rb, cuda, t, T, Hkv, Dh, page, gs):
    import torch
    g = torch.Generator("cuda").manual_seed(T)
    pages = -(-T // page) + 2
    gk, gv = ((0.25 * 2.0 ** torch.randint(0, 4, (Hkv,), generator=g, device="cuda")).float() for _ in range(2))
    cache = rb.KV4Cache.empty(pages, Hkv, page, Dh, gk if gs else None, gv if gs else None)
    one = torch.ones(Hkv, device="cuda")
    gk, gv = (gk, gv) if gs else (one, one)
    big = torch.randn(T, 2, Hkv, Dh, generator=g, device="cuda") * torch.exp(
        3 * torch.randn(T, 2, Hkv, 1, generator=g, device="cuda"))
    big[0, 0, 0, :16] = 0  # an empty block
    big = big.to(_dt(t))
    K, V = big[:, 0], big[:, 1]  # (strided tokens)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T].int()
    if T > 4:
        slots[2] = -1
    rb.kv4_write(cache, K, V, slots)
    rb.sync_status()
    keep = slots >= 0
    pg, at = slots[keep].long() // page, slots[keep].long() % page
    used = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    used[pg, at] = True
    k2, v2 = torch.full_like(K, 9).contiguous(), torch.full_like(V, 9).contiguous()
    rb.kv4_read(cache, slots, k2, v2)
    rb.sync_status()
    for x, codes, scales, gg, back in ((K, cache.tensors[0], cache.tensors[1], gk, k2),
                                       (V, cache.tensors[2], cache.tensors[3], gv, v2)):
        c, s = _quantize(x[keep], gg[None, :, None])
        assert torch.equal(codes[pg, :, at], c) and torch.equal(scales[pg, :, at], s)
        assert (codes.transpose(1, 2)[~used] == 0).all() and (scales.transpose(1, 2)[~used] == 0).all()
        want = _decode(codes, scales, gg)[pg, :, at]
        assert torch.equal(back[keep], want.float().to(_dt(t)))
        assert (back[~keep] == 9).all()


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shift,pad", [(0, 0), (16, 0), (0, 16), (16, 16), (32, 32)])
def test_write_and_read_on_16_byte_boundaries(rb, cuda, t, shift, pad):
    """Tokens at any multiple of 16 bytes, K's and V's independently: the codes and values of aligned ones,
    and nothing written between the rows."""
    import torch
    T, Hkv, Dh, page = 37, 3, 48, 16
    dt, es = _dt(t), torch.empty((), dtype=_dt(t)).element_size()
    x = torch.randn(T, Hkv, Dh, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(dt)
    slots = torch.arange(T, dtype=torch.int32, device="cuda")

    def view(fill):
        buf = torch.full(((shift + T * (Hkv * Dh * es + pad)) // es,), fill, dtype=dt, device="cuda")
        return buf, buf[shift // es:].as_strided((T, Hkv, Dh), (Hkv * Dh + pad // es, Dh, 1), shift // es)

    aligned, moved = (rb.KV4Cache.empty(3, Hkv, page, Dh) for _ in range(2))
    rb.kv4_write(aligned, x, x, slots)
    _, y = view(0)
    y.copy_(x)
    rb.kv4_write(moved, y, x, slots)
    for a, b in zip(aligned.tensors[:4], moved.tensors[:4]):
        assert torch.equal(a, b)
    want, other = torch.empty_like(x), torch.empty_like(x)
    rb.kv4_read(aligned, slots, want, other)
    buf, z = view(7)
    rb.kv4_read(aligned, slots, other, z)
    rb.sync_status()
    assert torch.equal(z, want) and torch.equal(other, want)
    z.fill_(7)
    assert (buf == 7).all()


def test_write_ties_and_specials(rb, cuda):
    """Every border between two codes, saturation, signed zeros, NaN and infinities, subnormal and huge scales."""
    import torch
    cache = rb.KV4Cache.empty(2, 1, 16, 64)
    K = torch.zeros(6, 1, 64, device="cuda")
    K[0, 0, :16] = torch.tensor([6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5, -.2])
    K[0, 0, 16:32] = 3 * K[0, 0, :16]
    K[1, 0, :16] = torch.tensor([float("nan"), 1, -1, 0.5, 2, -6] + [0.0] * 10)
    K[2, 0, :16] = torch.tensor([float("inf"), -float("inf"), 448 * 6, 448 * 3, -448, 1] + [-0.0] * 10)
    K[3, 0, :16] = 1e-4 * torch.arange(16)   # a subnormal e4m3 scale
    K[4, 0, :16] = 1e30
    K[4, 0, 16:32] = 1e-6                    # rounds to a zero scale
    K[5, 0, :] = float("nan")
    for t in ("f32", "bf16"):
        x = K.to(_dt(t))
        rb.kv4_write(cache, x, x, torch.arange(6, dtype=torch.int32, device="cuda"))
        rb.sync_status()
        c, s = _quantize(x, torch.ones(1, 1, 1, device="cuda"))
        got = cache.tensors[0][0, 0, :6], cache.tensors[1][0, 0, :6]
        assert torch.equal(got[1], s[:, 0])
        live = torch.tensor([0, 1, 2, 3, 4], device="cuda")  # (row 5: no scale, zero codes)
        assert torch.equal(got[0][live], c[live, 0])
        assert (got[0][5] == 0).all() and (got[1][5] == 0).all()


def test_attention_without_queries(rb, cuda):
    import torch
    cache = rb.KV4Cache.empty(2, 1, 16, 64)
    z = torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.empty(0, 4, 64, device="cuda")
    o = rb.attention_kv4(q, cache, z[:2], torch.zeros(2, 1, dtype=torch.int32, device="cuda"), cu_q=z)
    rb.sync_status()
    assert o.shape == q.shape


def test_bad_slots_are_reported(rb, cuda):
    import torch
    cache = rb.KV4Cache.empty(2, 2, 16, 32)
    K = torch.ones(3, 2, 32, device="cuda")
    slots = torch.tensor([0, 32, 2147483647], dtype=torch.int32, device="cuda")
    rb.kv4_write(cache, K, K, slots)
    with pytest.raises(rb.RougeB200Error) as e:
        rb.sync_status()
    assert e.value.status == rb.EINVAL
    assert (cache.tensors[1].transpose(1, 2).reshape(32, -1)[0] != 0).all()
    assert (cache.tensors[1].transpose(1, 2).reshape(32, -1)[1:] == 0).all()
    back = torch.full_like(K, 5)
    rb.kv4_read(cache, slots, back, back.clone())
    with pytest.raises(rb.RougeB200Error):
        rb.sync_status()
    # 1/6 rounds to the e4m3 value 11/64, and 1 / (11/64) = 5.8 to the code of 6
    assert (back[1:] == 5).all() and (back[0] == 66 / 64).all()
    rb.kv4_write(cache, K[:0], K[:0], slots[:0])
    rb.sync_status()


# ------------------------------------------------------------------ attention

@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("Hq,Hkv,Dh,page", [(4, 1, 16, 16), (8, 2, 48, 32), (8, 8, 64, 16), (14, 2, 80, 48),
                                            (6, 2, 96, 16), (8, 1, 128, 64), (16, 1, 128, 16), (40, 2, 112, 32),
                                            (4, 2, 192, 16), (9, 1, 256, 128)])
def test_decode(rb, cuda, t, Hq, Hkv, Dh, page):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 64, 100, 257, 0]
    cache = _cache(rb, sum(-(-n // page) for n in lens) + 1, Hkv, page, Dh, Hq + Dh)
    O = _check(rb, cache, t, lens, [1] * len(lens), Hq)
    assert (O[-1] == 0).all()


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("lens,Hq,Hkv,Dh", [([3000], 8, 1, 128), ([1, 5000, 40, 1023], 8, 2, 64), ([70001], 4, 1, 128),
                                            ([2049, 2048, 2047], 12, 3, 256)])
def test_long_sequences_are_split_and_joined(rb, cuda, t, lens, Hq, Hkv, Dh):
    cache = _cache(rb, sum(-(-n // 64) for n in lens) + 1, Hkv, 64, Dh, 3)
    _check(rb, cache, t, lens, [1] * len(lens), Hq)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("window", [0, 1, 7, 100])
def test_queries_and_windows(rb, cuda, t, causal, window):
    """Ragged numbers of queries: none, one, many, more than keys (those before the first key are empty rows)."""
    lens, nqs = [40, 5, 200, 33, 0, 130], [3, 9, 1, 33, 2, 0]
    for Hq, Hkv, Dh in ((6, 2, 64), (5, 1, 80)):
        cache = _cache(rb, 40, Hkv, 16, Dh, window)
        _check(rb, cache, t, lens, nqs, Hq, causal, window, extra=3)


@pytest.mark.parametrize("nq,n", [(17, 17), (64, 300), (150, 151), (129, 129)])
@pytest.mark.parametrize("t,Hq,Hkv,Dh", [("bf16", 8, 2, 128), ("f16", 3, 1, 64), ("f32", 4, 4, 64), ("bf16", 2, 1, 256)])
def test_prompt_chunks(rb, cuda, nq, n, t, Hq, Hkv, Dh):
    cache = _cache(rb, 2 * (-(-n // 32)) + 2, Hkv, 32, Dh, nq, gs=False)
    _check(rb, cache, t, [n, n - 1 if n > nq else n], [nq, nq], Hq)
    _check(rb, cache, t, [n], [nq], Hq, window=20)


@pytest.mark.parametrize("causal,window", [(1, 0), (0, 0), (1, 150), (0, 1)])
@pytest.mark.parametrize("t,Hq,Hkv,Dh,page", [("bf16", 16, 4, 128, 64), ("f16", 9, 3, 64, 16), ("bf16", 24, 8, 128, 48),
                                              ("bf16", 64, 1, 64, 32)])
def test_long_prompt_chunks(rb, cuda, t, Hq, Hkv, Dh, page, causal, window):
    """Enough rows for the kernel of 256-row tiles: ragged numbers of queries, more queries than keys, none, one."""
    lens, nqs = [700, 130, 64, 290, 5], [301, 130, 200, 0, 1]
    nqs = [n * 2 for n in nqs] if Hq == 9 else nqs
    cache = _cache(rb, sum(-(-n // page) for n in lens) + 1, Hkv, page, Dh, Hq, gs=window == 0)
    _check(rb, cache, t, lens, nqs, Hq, causal, window, extra=2, tiny_step=2.0 ** -32)


def test_long_chunks_masked_nan_bad_pages_and_same_bits(rb, cuda):
    import torch
    page, lens, nqs, window = 16, [400, 260], [256, 256], 70
    cache = _cache(rb, 60, 2, page, 128, 4)
    ids = torch.randperm(60).tolist()
    table = torch.full((2, 25), 1 << 30, dtype=torch.int32, device="cuda")
    seen = torch.zeros(60, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            table[b, i] = ids.pop()
        for k in range(max(0, n - nqs[b] - window + 1), n):
            seen[table[b, k // page].item(), k % page] = True
    args = ("bf16", lens, nqs, 32)
    clean = _check(rb, cache, *args, window=window, table=table, tiny_step=2.0 ** -32)
    for s in (cache.tensors[1], cache.tensors[3]):
        s.transpose(1, 2)[~seen.cuda()] = 0x7F
    _, O, *_ = _attend(rb, cache, *args, window=window, table=table)
    rb.sync_status()
    assert torch.equal(O, clean)
    table[0, 0] = -1  # wholly before the first query's window
    _, O, *_ = _attend(rb, cache, *args, window=window, table=table)
    rb.sync_status()
    assert torch.equal(O, clean)
    table[0, 20] = 60  # a page that a query needs
    _, O, *_ = _attend(rb, cache, *args, window=window, table=table)
    with pytest.raises(rb.RougeB200Error) as e:
        rb.sync_status()
    assert e.value.status == rb.EINVAL
    assert torch.equal(O[nqs[0]:], clean[nqs[0]:]) and O.isfinite().all()


def test_long_chunks_growing_scores(rb, cuda):
    """Keys whose scores grow along the sequence: the running maximum moves in every block of keys."""
    import torch
    cache = rb.KV4Cache.empty(20, 4, 64, 128)
    g = torch.Generator("cuda").manual_seed(2)
    n, nq = 1280, 400
    x = torch.randn(1, 4, 128, generator=g, device="cuda")
    K = x * torch.linspace(0.1, 4, n, device="cuda")[:, None, None] + 0.3 * torch.randn(n, 4, 128, generator=g, device="cuda")
    V = torch.randn(n, 4, 128, generator=g, device="cuda")
    rb.kv4_write(cache, K, V, torch.arange(n, dtype=torch.int32, device="cuda"))
    table = torch.arange(20, dtype=torch.int32, device="cuda")[None].contiguous()
    q = (1.5 * x.repeat_interleave(4, 1) + 0.3 * torch.randn(nq, 16, 128, generator=g, device="cuda")).bfloat16()
    lens, cu = torch.tensor([n], dtype=torch.int32, device="cuda"), torch.tensor([0, nq], dtype=torch.int32, device="cuda")
    O = rb.attention_kv4(q, cache, lens, table, cu_q=cu, max_q=nq)
    rb.sync_status()
    want, spread, ds, tiny = _reference(cache, q, [n], table, [nq], 1, 0, 128 ** -0.5, 2.0 ** -32)
    tol = (2 * ds + 2.0 ** -11 + 2.0 ** -21 + 200 * 2.0 ** -23) * spread + tiny
    tol = tol + _half_step(want.abs() + tol, q.dtype)
    assert ((O.double() - want).abs() <= tol).all()


def test_scale_argument_and_wide_values(rb, cuda):
    """Queries whose rows differ by 2^40 and a large scale: the row's power of two keeps f16 operands in range."""
    import torch
    cache = _cache(rb, 20, 2, 16, 64, 8)
    g = torch.Generator("cuda").manual_seed(1)
    lens = torch.tensor([250, 30], dtype=torch.int32, device="cuda")
    table = torch.arange(32, dtype=torch.int32, device="cuda").reshape(2, 16) % 20
    q = torch.randn(2, 4, 64, generator=g, device="cuda") * torch.tensor([1e-12, 1e-3, 1.0, 1e5], device="cuda")[:, None]
    for t in ("f32", "bf16"):
        qq = q.to(_dt(t))
        O = rb.attention_kv4(qq, cache, lens, table, scale=1e-5)
        rb.sync_status()
        want, spread, ds, tiny = _reference(cache, qq, [250, 30], table, [1, 1], 1, 0, 1e-5)
        w = 2.0 ** -21 + (2.0 ** -21 if t == "f32" else 2.0 ** -11)
        tol = (2 * ds + w + 80 * 2.0 ** -23) * spread + tiny
        tol = tol + _half_step(want.abs() + tol, qq.dtype)
        assert ((O.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_what_is_masked_is_not_read_into_results(rb, cuda, t):
    """NaN scales in every slot that no query may see: past the length, before the window, in unused pages."""
    import torch
    page, lens, window = 16, [37, 90, 16], 21
    cache = _cache(rb, 16, 2, page, 64, 4)
    table = torch.full((3, 6), 1 << 30, dtype=torch.int32, device="cuda")
    ids = torch.randperm(16).tolist()
    seen = torch.zeros(16, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            table[b, i] = ids.pop()
        for k in range(max(0, n - window), n):
            seen[table[b, k // page].item(), k % page] = True
    kc, ks, vc, vs, _, _ = cache.tensors
    clean = _check(rb, cache, t, lens, [1, 1, 1], 4, window=window, table=table)
    for s in (ks, vs):
        s.transpose(1, 2)[~seen.cuda()] = 0x7F
    q, O, *_ = _attend(rb, cache, t, lens, [1, 1, 1], 4, window=window, table=table)
    rb.sync_status()
    assert torch.equal(O, clean)
    table[1, 0] = -1  # a page wholly before the window may be gone
    _, O, *_ = _attend(rb, cache, t, lens, [1, 1, 1], 4, window=window, table=table)
    rb.sync_status()
    assert torch.equal(O, clean)


def test_bad_pages_are_reported_and_taken_as_masked(rb, cuda):
    import torch
    cache = _cache(rb, 8, 1, 16, 64, 2)
    table = torch.arange(8, dtype=torch.int32, device="cuda").reshape(2, 4)
    lens = torch.tensor([64, 50], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 64, device="cuda")
    good = rb.attention_kv4(q, cache, lens, table)
    rb.sync_status()
    for bad in (-1, 8, 2147483647, -2147483648):
        broken = table.clone()
        broken[0, 1] = bad
        O = rb.attention_kv4(q, cache, lens, broken)
        with pytest.raises(rb.RougeB200Error) as e:
            rb.sync_status()
        assert e.value.status == rb.EINVAL
        assert torch.equal(O[1], good[1]) and O.isfinite().all()
    # a length past the table: the keys that have a page count
    for n in (1000, 2147483647):
        O = rb.attention_kv4(q, cache, torch.tensor([n, 50], dtype=torch.int32, device="cuda"), table)
        with pytest.raises(rb.RougeB200Error):
            rb.sync_status()
        assert torch.equal(O[1], good[1]) and (O[0] - good[0]).abs().max() < 1e-5
    # a negative one is none
    O = rb.attention_kv4(q, cache, torch.tensor([-5, 50], dtype=torch.int32, device="cuda"), table)
    assert torch.equal(O[1], good[1]) and (O[0] == 0).all()
    # a window past every distance hides nothing
    assert torch.equal(rb.attention_kv4(q, cache, lens, table, window=2147483647), good)
    rb.sync_status()


@pytest.mark.parametrize("B", [33, 100, 700])
def test_many_sequences(rb, cuda, B):
    """More sequences than a warp holds at a time, empty and one-key ones among them."""
    lens = [(7 * b) % 90 for b in range(B)]
    nqs = [(b % 5 != 3) * (1 + (b % 7 == 0)) for b in range(B)]
    cache = _cache(rb, sum(-(-n // 16) for n in lens) + 1, 2, 16, 64, B)
    _check(rb, cache, "bf16", lens, nqs, 6, extra=1)
    _check(rb, cache, "f32", lens, [1] * B, 2)


def test_same_call_same_bits_and_shared_pages(rb, cuda):
    import torch
    cache = _cache(rb, 70, 2, 64, 128, 6)
    table = torch.arange(70, dtype=torch.int32, device="cuda").repeat(3, 1)  # (three sequences on the same pages)
    lens = [4400, 4480, 1000]
    q, O, _, lens_d, _ = _attend(rb, cache, "bf16", lens, [1, 1, 1], 16, table=table)
    for _ in range(5):
        assert torch.equal(rb.attention_kv4(q, cache, lens_d, table), O)
    rb.sync_status()


def test_captured_replayed_and_on_another_stream(rb, cuda):
    """One capture serves growing lengths; two streams at a time need two workspaces."""
    import torch
    cache = _cache(rb, 64, 2, 32, 64, 5)
    table = torch.arange(64, dtype=torch.int32, device="cuda").reshape(2, 32)
    q = torch.randn(2, 8, 64, device="cuda").bfloat16()
    lens = torch.tensor([3, 40], dtype=torch.int32, device="cuda")
    n = rb.attention_kv4_workspace(2, 8, 2, 64, 1, 1024, rb.T_BF16)
    ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in range(2)]
    out = torch.empty_like(q)
    rb.attention_kv4(q, cache, lens, table, O=out, workspace=ws[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rb.attention_kv4(q, cache, lens, table, O=out, workspace=ws[0])
    side = torch.cuda.Stream()
    for a, b in ((3, 40), (1000, 1024), (0, 1)):
        lens.copy_(torch.tensor([a, b]))
        want = rb.attention_kv4(q, cache, lens, table)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other = rb.attention_kv4(q, cache, lens, table, workspace=ws[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(other, want)
    rb.sync_status()


def test_workspace_is_checked(rb, cuda):
    import torch
    cache = _cache(rb, 4, 1, 16, 64, 5)
    q, lens = torch.randn(1, 2, 64, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    table = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    n = rb.attention_kv4_workspace(1, 2, 1, 64, 1, 64, rb.T_F32)
    with pytest.raises(rb.RougeB200Error) as e:
        rb.attention_kv4(q, cache, lens, table, workspace=torch.empty(n - 1, dtype=torch.uint8, device="cuda"))
    assert e.value.status == rb.ETOOBIG


def test_decoder_step_together(rb, cuda):
    """norm -> int8 QKV product with bias -> cache write -> attention over the cache -> output product with the
    residual, three tokens in a row, against the same steps in f32 / 64 bits from the intermediate codes."""
    import torch
    g = torch.Generator("cuda").manual_seed(0)
    B, D, Hq, Hkv, Dh, page = 5, 256, 8, 2, 64, 16
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    N = (Hq + 2 * Hkv) * Dh
    wqkv, wo, bias, wn = rn(N, D) / 16, rn(D, Hq * Dh) / 23, rn(N), 0.5 + torch.rand(D, generator=g, device="cuda")

    def q8(w):
        q, s = torch.empty(w.shape, dtype=torch.int8, device="cuda"), torch.empty(w.shape[0], device="cuda")
        rb.quantize_i8_rows(w.contiguous(), s, q)
        return q, s
    qkv_q, qkv_s = q8(wqkv)
    o_q, o_s = q8(wo)
    cache = rb.KV4Cache.empty(8, Hkv, page, Dh)
    table = torch.arange(B, dtype=torch.int32, device="cuda")[:, None].contiguous()
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    res = rn(B, D).bfloat16()
    for step in range(3):
        x = rn(B, D).bfloat16()
        h, codes, scales = torch.empty_like(x), torch.empty(B, D, dtype=torch.int8, device="cuda"), torch.empty(
            B, device="cuda")
        rb.add_rmsnorm_quant(x, res, wn, 1e-5, rb.Q_I8_ROWS, codes, scales, h)
        qkv = torch.empty(B, N, dtype=torch.bfloat16, device="cuda")
        rb.gemm_i8(codes, qkv_q, rb.B_NK, qkv, rb.OUT_BF16, scales, 1, qkv_s, 1, epilogue=rb.Epilogue(bias))
        q = qkv[:, :Hq * Dh].reshape(B, Hq, Dh).contiguous()
        k, v = qkv[:, Hq * Dh:(Hq + Hkv) * Dh].unflatten(1, (Hkv, Dh)), qkv[:, (Hq + Hkv) * Dh:].unflatten(1, (Hkv, Dh))
        rb.kv4_write(cache, k, v, table[:, 0] * page + lens)
        lens += 1
        att = rb.attention_kv4(q, cache, lens, table)
        aq, asc = q8(att.reshape(B, Hq * Dh).float())
        out = h.clone()
        rb.gemm_i8(aq, o_q, rb.B_NK, out, rb.OUT_BF16, asc, 1, o_s, 1, epilogue=rb.Epilogue(residual=out))
        rb.sync_status()
        # each step from the one before it
        want_h = (x.float() + res.float()).bfloat16()
        assert torch.equal(h, want_h)
        wq = (codes.double() @ qkv_q.double().T) * scales.double()[:, None] * qkv_s.double() + bias.double()
        assert ((qkv.double() - wq).abs() <= wq.abs() * 2.0 ** -8 + 2.0 ** -20).all()
        ref, spread, ds, _ = _reference(cache, q, [step + 1] * B, table, [1] * B, 1, 0, 1 / 8)
        assert ((att.double() - ref).abs() <= (2 * ds + 2.0 ** -10) * spread + ref.abs() * 2.0 ** -8).all()
        wo_ = (aq.double() @ o_q.double().T) * asc.double()[:, None] * o_s.double() + h.double()
        assert ((out.double() - wo_).abs() <= wo_.abs() * 2.0 ** -8 + 2.0 ** -20).all()
        res = out


def _sequence_reference(cache, q, n, row, window, hidden, tiny_step):
    """O and the tolerance's parts of one causal sequence in 64 bits, without its keys t where hidden[t]."""
    import torch
    kc, ks, vc, vs, gk, gv = cache.tensors
    one = torch.ones(cache.Hkv, device="cuda")
    nq, G = q.shape[0], q.shape[1] // cache.Hkv
    t = torch.arange(n, device="cuda")
    pg, off = row.long().clamp(0, cache.pages - 1)[t // cache.page], t % cache.page
    K = _decode(kc, ks, gk if gk is not None else one)[pg, :, off].repeat_interleave(G, 1)
    V = _decode(vc, vs, gv if gv is not None else one)[pg, :, off].repeat_interleave(G, 1)
    p = n - nq + torch.arange(nq, device="cuda")[:, None]
    ok = (t <= p) & ~hidden & ((t > p - window) if window else True)
    scale = cache.Dh ** -0.5
    z = torch.einsum("ihd,thd->hit", q.double(), K) * scale
    za = torch.einsum("ihd,thd->hit", q.double().abs(), K.abs()) * scale
    w = torch.softmax(z.masked_fill(~ok, -math.inf), -1).nan_to_num(0)  # (a row without keys)
    ds = (za.masked_fill(~ok, 0).amax(-1) * (cache.Dh / 16 + 6) * 2.0 ** -23).T[..., None]
    return (torch.einsum("hit,thd->ihd", w, V), torch.einsum("hit,thd->ihd", w, V.abs()), ds,
            tiny_step * torch.einsum("it,thd->ihd", ok.double(), V.abs()))


def _close(O, want, spread, ds, tiny, t, n):
    w = 2.0 ** -21 + (2.0 ** -21 if t == "f32" else 2.0 ** -11)
    tol = (2 * ds + w + (max(n, 16) / 16 + 64) * 2.0 ** -23) * spread + tiny
    tol = tol + _half_step(want.abs() + tol, O.dtype)
    d = (O.double() - want).abs()
    assert (d <= tol).all(), ((d / tol.clamp(min=1e-300)).nan_to_num(math.inf).max().item(), d.max().item())


@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("t,nq,Hq,Dh", [("f32", 1, 4, 64), ("bf16", 1, 4, 128), ("f16", 20, 8, 80),
                                        ("bf16", 500, 16, 128), ("f16", 700, 16, 64)])
def test_keys_on_bad_pages_have_no_weight(rb, cuda, t, nq, Hq, Dh, window):
    """Scores far below zero: a key taken in with a score of zero would outweigh all others."""
    import torch
    Hkv, page, n = 4, 16, 730
    g = torch.Generator("cuda").manual_seed(nq + Dh)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    cache = rb.KV4Cache.empty(46, Hkv, page, Dh)
    x = rn(1, Hkv, Dh)
    rb.kv4_write(cache, -x + 0.3 * rn(n, Hkv, Dh), rn(n, Hkv, Dh), torch.arange(n, dtype=torch.int32, device="cuda"))
    q = (x.repeat_interleave(Hq // Hkv, 1) + 0.2 * rn(nq, Hq, Dh)).to(_dt(t))
    table = torch.arange(46, dtype=torch.int32, device="cuda")[None].clone()
    hidden = torch.zeros(n, dtype=torch.bool, device="cuda")
    for i, bad in ((0, -1), (14, 46), (15, 1 << 30), (41, -1 << 31), (45, 46)):
        table[0, i] = bad
        hidden[i * page:(i + 1) * page] = True
    cu = torch.tensor([0, nq], dtype=torch.int32, device="cuda")
    O = rb.attention_kv4(q, cache, torch.tensor([n], dtype=torch.int32, device="cuda"), table, cu_q=cu, max_q=nq,
                         window=window)
    with pytest.raises(rb.RougeB200Error) as e:
        rb.sync_status()
    assert e.value.status == rb.EINVAL
    tiny = 2.0 ** -32 if nq >= 500 else 2.0 ** -40
    _close(O, *_sequence_reference(cache, q, n, table[0], window, hidden, tiny), t, n)


@pytest.mark.parametrize("t,up", [("f32", 10), ("f32", 14), ("f32", 20), ("bf16", 14), ("bf16", 24), ("f16", 14)])
@pytest.mark.parametrize("nq,Hq,Dh", [(1, 4, 64), (1, 32, 128), (9, 4, 256), (400, 16, 128)])
def test_query_channels_far_above_the_others(rb, cuda, t, up, nq, Hq, Dh):
    """Two channels 2^up above the rest meet zero codes: the scores are those of the small channels, whose values
    are held to 2^-23 of their own size (16-bit queries exactly), not of the largest one's."""
    import torch
    n = 410
    cache = _cache(rb, 26, 4, 16, Dh, up)
    kc = cache.tensors[0]
    kc[..., 2] &= 0xF0       # channel 4
    kc[..., Dh // 2 - 1] &= 0x0F  # channel Dh - 1
    g = torch.Generator("cuda").manual_seed(nq + Dh)
    q = torch.randn(nq, Hq, Dh, generator=g, device="cuda")
    q[..., 4], q[..., Dh - 1] = 1.37 * 2.0 ** up, -1.9 * 2.0 ** up
    q = q.to(_dt(t))
    table = torch.randperm(26, generator=g, device="cuda").int()[None]
    cu = torch.tensor([0, nq], dtype=torch.int32, device="cuda")
    O = rb.attention_kv4(q, cache, torch.tensor([n], dtype=torch.int32, device="cuda"), table, cu_q=cu, max_q=nq)
    rb.sync_status()
    hidden = torch.zeros(n, dtype=torch.bool, device="cuda")
    _close(O, *_sequence_reference(cache, q, n, table[0], 0, hidden, 2.0 ** -32 if nq == 400 else 2.0 ** -40), t, n)


@pytest.mark.parametrize("t,Hq,Dh,page,counts,max_q", [("f32", 4, 64, 16, [3, 5, 2], 3), ("bf16", 8, 80, 16, [3, 1, 2], 1),
                                                       ("bf16", 16, 128, 32, [300, 301, 7], 300)])
def test_queries_past_max_q_are_reported(rb, cuda, t, Hq, Dh, page, counts, max_q):
    """They are left as they were; the others keep their positions and values."""
    import torch
    n, Hkv, T = 320, 4, sum(counts)
    cache = _cache(rb, 3 * n // page, Hkv, page, Dh, max_q)
    table = torch.arange(3 * n // page, dtype=torch.int32, device="cuda").reshape(3, -1)
    lens = torch.full((3,), n, dtype=torch.int32, device="cuda")
    cu = torch.tensor(np.concatenate(([0], np.cumsum(counts))), dtype=torch.int32, device="cuda")
    q = torch.randn(T, Hq, Dh, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(_dt(t))
    want = rb.attention_kv4(q, cache, lens, table, cu_q=cu, max_q=max(counts))
    rb.sync_status()
    O = torch.full_like(q, 77.0)
    rb.attention_kv4(q, cache, lens, table, cu_q=cu, max_q=max_q, O=O)
    with pytest.raises(rb.RougeB200Error) as e:
        rb.sync_status()
    assert e.value.status == rb.EINVAL
    done = torch.cat([torch.arange(c, device="cuda") < max_q for c in counts])
    assert (O[~done] == 77).all()
    # (another max_q may take another kernel: equal up to both kernels' roundings of weights and output)
    assert torch.allclose(O[done].float(), want[done].float(), rtol=0, atol=2.0 ** -6)


@pytest.mark.parametrize("t,Hq,Dh,max_q", [("f32", 4, 64, 3), ("bf16", 16, 128, 400)])
def test_query_offsets_that_fall_are_reported(rb, cuda, t, Hq, Dh, max_q):
    """Sequences whose offsets fall or are negative are left out; the others are computed."""
    import torch
    cache = _cache(rb, 40, 4, 16, Dh, 2)
    table = torch.arange(40, dtype=torch.int32, device="cuda").reshape(4, 10)
    lens = torch.full((4,), 160, dtype=torch.int32, device="cuda")
    q = torch.randn(9, Hq, Dh, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(_dt(t))
    run = lambda cu, O: rb.attention_kv4(q, cache, lens, table, max_q=max_q, O=O,  # noqa: E731
                                         cu_q=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    want = run([0, 3, 3, 3, 6], torch.full_like(q, 77.0))
    rb.sync_status()
    for cu in ([0, 3, 1, 3, 6], [-2, 0, 3, 3, 6], [-2147483648, 0, 3, 3, 6], [2147483647, 0, 3, 3, 6]):
        O = run(cu, torch.full_like(q, 77.0))
        with pytest.raises(rb.RougeB200Error) as e:
            rb.sync_status()
        assert e.value.status == rb.EINVAL
        assert torch.equal(O[3:], want[3:])


def test_workspace_does_not_depend_on_the_sm_budget(rb, cuda):
    """Sized under one budget of SMs and used under another."""
    import torch
    cache = _cache(rb, 200, 2, 16, 64, 5)
    q = torch.randn(3, 8, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    lens = torch.tensor([1000, 3, 1056], dtype=torch.int32, device="cuda")
    table = torch.arange(198, dtype=torch.int32, device="cuda").reshape(3, 66)
    size = lambda: rb.attention_kv4_workspace(3, 8, 2, 64, 1, 1056, rb.T_F32)  # noqa: E731
    n = size()
    L = rb.lib()
    old = L.rouge_b200_set_sm_budget(5)
    try:
        small = size()
        assert small == n
        ws = torch.empty(small, dtype=torch.uint8, device="cuda")
        few = rb.attention_kv4(q, cache, lens, table, workspace=ws).clone()
    finally:
        L.rouge_b200_set_sm_budget(old)
    all_ = rb.attention_kv4(q, cache, lens, table, workspace=ws)
    rb.sync_status()
    want, spread, ds, tiny = _reference(cache, q, [1000, 3, 1056], table, [1, 1, 1], 1, 0, 1 / 8)
    _close(few, want, spread, ds, tiny, "f32", 1056)
    _close(all_, want, spread, ds, tiny, "f32", 1056)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("g", [2.0 ** -10, 1e-30, 1e20])
def test_write_saturates_with_the_sign(rb, cuda, t, g):
    """Values so far above 448 * 6 * gs that their quotient by the block's step leaves f32's range."""
    import torch
    gs = torch.tensor([g], device="cuda")
    cache = rb.KV4Cache.empty(1, 1, 16, 32, gs, gs)
    top = torch.finfo(torch.bfloat16).max
    K = torch.zeros(3, 1, 32, device="cuda")
    K[0, 0, :8] = torch.tensor([top, -top, top / 2, -top / 2, 1.0, -1.0, -1e30, 1e30])
    K[1, 0, 16:20] = torch.tensor([-top, 3 * g, -6 * 448 * g, 448 * g])
    K[2, 0, :4] = torch.tensor([-1e9, 1e9, -1e-3, 0.0])
    x = K.to(_dt(t))
    rb.kv4_write(cache, x, x, torch.arange(3, dtype=torch.int32, device="cuda"))
    rb.sync_status()
    c, s = _quantize(x, gs[None, :, None])
    for codes, scales in (cache.tensors[:2], cache.tensors[2:4]):
        assert torch.equal(scales[0, 0, :3], s[:, 0]) and torch.equal(codes[0, 0, :3], c[:, 0])


@pytest.mark.parametrize("B,nq", [(1, 1), (5, 1), (5, 3), (300, 1), (40, 20)])
def test_workspace_needs_no_initialisation(rb, cuda, B, nq):
    """Whatever bytes it holds, also for sequences without queries, whose units nothing writes."""
    import torch
    g = torch.Generator("cuda").manual_seed(B)
    cache = _cache(rb, 128, 2, 16, 64, B)
    lens = torch.randint(0, 2049, (B,), generator=g, device="cuda").int()
    table = torch.randint(0, 128, (B, 128), generator=g, device="cuda").int()
    counts = torch.randint(0, nq + 1, (B,), generator=g, device="cuda") if nq > 1 else torch.ones(B, device="cuda")
    cu = torch.cat((torch.zeros(1, device="cuda"), counts.cumsum(0))).int()
    q = torch.randn(B * nq, 8, 64, generator=g, device="cuda").bfloat16()
    ws = torch.zeros(rb.attention_kv4_workspace(B, 8, 2, 64, nq, 2048, rb.T_BF16), dtype=torch.uint8, device="cuda")
    outs = []
    for fill in (0, 0x7F, 0xFF, 0x01):
        ws.fill_(fill)
        O = torch.full_like(q, 77.0)
        rb.attention_kv4(q, cache, lens, table, cu_q=cu, max_q=nq, O=O, workspace=ws)
        rb.sync_status()
        outs.append(O)
    assert all(torch.equal(o, outs[0]) for o in outs) and (outs[0][cu[-1]:] == 77).all()
    assert outs[0].isfinite().all()


@pytest.mark.parametrize("t,nq,Hq", [("f32", 1, 4), ("bf16", 3, 8), ("bf16", 500, 16)])
def test_window_counts_from_the_length_past_the_table(rb, cuda, t, nq, Hq):
    """A length past the table's 640 keys (reported): those with a page are visible where the window reaches them."""
    import torch
    n, have, window = 1100, 640, 700
    cache = _cache(rb, 40, 4, 16, 64, 3)
    table = torch.arange(40, dtype=torch.int32, device="cuda")[None]
    q = torch.randn(nq, Hq, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(nq)).to(_dt(t))
    O = rb.attention_kv4(q, cache, torch.tensor([n], dtype=torch.int32, device="cuda"), table, max_q=nq, window=window,
                         cu_q=torch.tensor([0, nq], dtype=torch.int32, device="cuda"))
    with pytest.raises(rb.RougeB200Error):
        rb.sync_status()
    longer = torch.cat((table, torch.zeros(1, n // 16, dtype=torch.int32, device="cuda")), 1)
    hidden = torch.arange(n, device="cuda") >= have
    _close(O, *_sequence_reference(cache, q, n, longer[0], window, hidden, 2.0 ** -32 if nq == 500 else 2.0 ** -40), t,
           have)


@pytest.mark.parametrize("t,nq,Hq,Dh", [("f32", 1, 8, 64), ("bf16", 1, 8, 128), ("f16", 7, 8, 96), ("bf16", 500, 16, 128)])
def test_special_queries_stay_in_their_rows(rb, cuda, t, nq, Hq, Dh):
    """NaN and infinities in some heads' queries: those rows are NaN, the others as without them."""
    import torch
    n = 520
    cache = _cache(rb, 33, 4, 16, Dh, nq)
    g = torch.Generator("cuda").manual_seed(nq)
    table = torch.randperm(33, generator=g, device="cuda").int()[None]
    q = torch.randn(nq, Hq, Dh, generator=g, device="cuda").to(_dt(t))
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, nq], dtype=torch.int32, device="cuda")
    run = lambda x: rb.attention_kv4(x, cache, lens, table, cu_q=cu, max_q=nq)  # noqa: E731
    good = run(q)
    odd = q.clone()
    odd[0, 0, 3], odd[nq // 2, 5, Dh - 1], odd[nq - 1, 2, :] = math.nan, math.inf, -math.inf
    O = run(odd)
    rb.sync_status()
    hit = torch.zeros(nq, Hq, dtype=torch.bool, device="cuda")
    hit[0, 0] = hit[nq // 2, 5] = hit[nq - 1, 2] = True
    assert O[hit].isnan().all() and torch.equal(O[~hit], good[~hit])


def test_decoder_step_in_f32(rb, cuda):
    """The chain with f32 queries, keys and values, which quantize_i8_rows takes from the attention as they are."""
    import torch
    g = torch.Generator("cuda").manual_seed(1)
    T, D, Hq, Hkv, Dh, page = 9, 512, 8, 2, 64, 16
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    i8 = lambda *s: torch.empty(*s, dtype=torch.int8, device="cuda")  # noqa: E731
    N = (Hq + 2 * Hkv) * Dh

    def q8(w):
        q, s = i8(*w.shape), torch.empty(w.shape[0], device="cuda")
        rb.quantize_i8_rows(w.contiguous(), s, q)
        return q, s
    (wqkv, sw), (wo, swo) = q8(rn(N, D) / 23), q8(rn(D, Hq * Dh) / 23)
    w, bias = 0.5 + torch.rand(D, generator=g, device="cuda"), rn(N)
    cache = rb.KV4Cache.empty(4, Hkv, page, Dh)
    x, r, h = rn(T, D).bfloat16(), rn(T, D).bfloat16(), torch.empty(T, D, dtype=torch.bfloat16, device="cuda")
    qx, sx = i8(T, D), torch.empty(T, device="cuda")
    rb.add_rmsnorm_quant(x, r, w, 1e-5, rb.Q_I8_ROWS, qx, sx, h)
    qkv = torch.empty(T, N, device="cuda")
    rb.gemm_i8(qx, wqkv, rb.B_NK, qkv, rb.OUT_F32, sx, 1, sw, 1, epilogue=rb.Epilogue(bias))
    k, v = (qkv[:, a * Dh:(a + Hkv) * Dh].unflatten(1, (Hkv, Dh)) for a in (Hq, Hq + Hkv))
    rb.kv4_write(cache, k, v, torch.arange(16, 16 + T, dtype=torch.int32, device="cuda"))
    q = qkv[:, :Hq * Dh].reshape(T, Hq, Dh).contiguous()
    table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    att = rb.attention_kv4(q, cache, torch.tensor([T], dtype=torch.int32, device="cuda"), table, max_q=T,
                           cu_q=torch.tensor([0, T], dtype=torch.int32, device="cuda"))
    o8, so = q8(att.reshape(T, Hq * Dh))
    out = h.clone()
    rb.gemm_i8(o8, wo, rb.B_NK, out, rb.OUT_BF16, so, 1, swo, 1, epilogue=rb.Epilogue(residual=out))
    rb.sync_status()
    wq = (qx.double() @ wqkv.double().T) * sx.double()[:, None] * sw.double()
    assert ((qkv.double() - wq - bias.double()).abs() <= 2.0 ** -22 * (wq.abs() + bias.double().abs())).all()
    hidden = torch.zeros(T, dtype=torch.bool, device="cuda")
    _close(att, *_sequence_reference(cache, q, T, table[0], 0, hidden, 2.0 ** -40), "f32", T)
    wo_ = (o8.double() @ wo.double().T) * so.double()[:, None] * swo.double() + h.double()
    assert ((out.double() - wo_).abs() <= wo_.abs() * 2.0 ** -8 + 2.0 ** -20).all()


def test_cache_offsets_past_32_bits(rb, cuda):
    """Pages whose codes lie past 2^32 bytes: written, read and attended to as the same tokens in a small cache."""
    import torch
    Hkv, page, Dh, pages, n = 8, 64, 128, 135000, 700   # 4.4 GB of codes each for keys and values
    big, small = rb.KV4Cache.empty(pages, Hkv, page, Dh), rb.KV4Cache.empty(12, Hkv, page, Dh)
    assert big.tensors[0].numel() > 1 << 32
    g = torch.Generator("cuda").manual_seed(7)
    K, V = (torch.randn(n, Hkv, Dh, generator=g, device="cuda").bfloat16() for _ in range(2))
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    per = -(-n // page)
    rb.kv4_write(small, K, V, at)
    rb.kv4_write(big, K, V, at + (pages - per) * page)
    outs = [torch.empty_like(K) for _ in range(4)]
    rb.kv4_read(small, at, *outs[:2])
    rb.kv4_read(big, at + (pages - per) * page, *outs[2:])
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
    low = torch.arange(per, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    for nq in (1, 5, 400):
        q = torch.randn(nq, 16, Dh, generator=g, device="cuda").bfloat16()
        cu = torch.tensor([0, nq], dtype=torch.int32, device="cuda")
        a, b = (rb.attention_kv4(q, c, lens, (low + first).contiguous(), cu_q=cu, max_q=nq)
                for c, first in ((small, 0), (big, pages - per)))
        assert torch.equal(a, b) and a.float().abs().max() > 0.01
    rb.sync_status()
