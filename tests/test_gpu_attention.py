"""GPU: the attention half served from the 8-bit cache (attention.py over
noor_rope_apply, noor_kv_append, noor_kv_read, noor_kv_attention) against its
plain 64-bit form (tests/attention_ref.py).

Tolerances, fixed before the first run:
  rotary      own rounding (BF16 2^-8, F32 2^-24 of the value) + 10 * 2^-24 (|x0| + |x1|) |factor|:
              the angle's fraction in f32 (3.2 units), sine and cosine (2), products and sum (3)
  cache       scales and codes equal; values read back equal (BF16 holds 8-bit codes times a power of two)
  attention   attention_ref.attend_tolerance
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests import attention_ref as ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
i32 = lambda xs: torch.tensor(xs, dtype=torch.int32, device="cuda")


def cu_of(counts):
    return i32([0] + np.cumsum(counts).tolist())


def randn(shape, seed, dtype=torch.float32, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * gain).to(dtype)


# ---------------------------------------------------------------- rotary


def check_rope(got, x, pos, inv, layout, factor, sign=1.0):
    want = ref.rotate(x, pos, inv, layout, factor, sign)
    own = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    half = inv.numel()
    pair = torch.zeros_like(want)
    if half:
        i0, i1 = ((torch.arange(half) * 2, torch.arange(half) * 2 + 1) if layout == "interleaved" else
                  (torch.arange(half), torch.arange(half) + half))
        pair[..., i0] = pair[..., i1] = x.double()[..., i0].abs() + x.double()[..., i1].abs()
    tol = own * want.abs() + 10 * 2.0 ** -24 * pair * abs(factor) * (1 + own) + 1e-38
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    assert torch.equal(got.cpu()[..., 2 * half:], x[..., 2 * half:].to(got.dtype))  # the rest passes unchanged


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("T,Hq,Hk,D,rot,start", [(1, 1, 0, 2, 2, 0), (1, 32, 8, 128, 128, 2 ** 31 - 1), (7, 4, 2, 64, 16, 10 ** 6),
                                                 (5, 3, 1, 80, 20, 77), (33, 2, 2, 48, 0, 5), (130, 9, 3, 256, 256, 131072),
                                                 (3, 2, 1, 18, 6, -9), (64, 1, 1, 1024, 1024, 4)])
def test_rope(pkg, cuda_device, dtype, layout, T, Hq, Hk, D, rot, start):
    A = pkg.attention
    inv = torch.from_numpy((10000.0 ** (-2.0 * np.arange(rot // 2) / max(rot, 1))).astype(np.float32))
    r = A.Rotary(inv.cuda(), layout, 1.25)
    pos = torch.clamp(torch.arange(T) + start, max=2 ** 31 - 1).to(torch.int32)
    q, k = randn((T, Hq, D), 1, DT[dtype]), randn((T, max(Hk, 1), D), 2, DT[dtype])
    if Hk:
        gq, gk = A.rope_apply(q.cuda(), pos.cuda(), r, k=k.cuda())
        check_rope(gk, k, pos, inv, layout, 1.25)
    else:
        gq = A.rope_apply(q.cuda(), pos.cuda(), r)
    check_rope(gq, q, pos, inv, layout, 1.25)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rope_views_and_unaligned(pkg, cuda_device, dtype):
    """q and k as slices of one fused tensor, heads outermost, a broadcast
    token and a base off by one element."""
    A = pkg.attention
    inv, _ = A.rotary_frequencies(64, 10000.0, 0.5)
    inv = torch.from_numpy(inv)
    r = A.Rotary(inv.numpy(), "half", device=0)
    T = 9
    pos = torch.randint(0, 50000, (T,), generator=torch.Generator().manual_seed(3)).to(torch.int32)
    fused = randn((T, 7, 64), 4, DT[dtype])
    f = fused.cuda()
    gq, gk = A.rope_apply(f[:, :4], pos.cuda(), r, k=f[:, 4:6])
    check_rope(gq, fused[:, :4], pos, inv, "half", 1.0)
    check_rope(gk, fused[:, 4:6], pos, inv, "half", 1.0)
    heads_first = f.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(A.rope_apply(heads_first, pos.cuda(), r), A.rope_apply(f, pos.cuda(), r))
    one = f[:1].expand(T, 7, 64)
    check_rope(A.rope_apply(one, pos.cuda(), r), fused[:1].expand(T, 7, 64), pos, inv, "half", 1.0)
    flat = torch.empty(T * 7 * 64 + 1, dtype=DT[dtype], device="cuda")
    off = flat[1:].view(T, 7, 64)
    off.copy_(f)
    check_rope(A.rope_apply(off, pos.cuda(), r), fused, pos, inv, "half", 1.0)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_gradient(pkg, cuda_device, layout):
    """The gradient is the transposed rotation; checked against the formula,
    against differences, and for gradients that arrive broadcast."""
    A = pkg.attention
    inv, factor = A.rotary_frequencies(32, 10000.0, 0.75, yarn={"scale": 4.0, "original": 2048})
    r = A.Rotary(inv, layout, factor)
    inv = torch.from_numpy(inv)
    pos = i32([5, 0, 4096])
    q, k = randn((3, 2, 32), 5).cuda().requires_grad_(), randn((3, 1, 32), 6).cuda().requires_grad_()
    wq, wk = randn((3, 2, 32), 7), randn((3, 1, 32), 8)
    oq, ok = A.rope_apply(q, pos, r, k=k)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (wq.cuda(), wk.cuda()))
    check_rope(dq, wq, pos.cpu(), inv, layout, factor, -1.0)
    check_rope(dk, wk, pos.cpu(), inv, layout, factor, -1.0)
    # differences of sum(w . rope(q)): linear in q, so a step of 1/2 is exact but for rounding
    e = randn((3, 2, 32), 9)
    f = lambda x: float((ref.rotate(x, pos.cpu(), inv, layout, factor) * wq.double()).sum())
    slope = (f(q.detach().cpu().double() + 0.5 * e.double()) - f(q.detach().cpu().double() - 0.5 * e.double()))
    assert abs(slope - float((dq.cpu().double() * e.double()).sum())) <= 1e-5 * 3 * 2 * 32
    (g,) = torch.autograd.grad(A.rope_apply(q, pos, r).sum(), q)  # an expanded gradient
    check_rope(g, torch.ones((3, 2, 32)), pos.cpu(), inv, layout, factor, -1.0)
    (g,) = torch.autograd.grad(A.rope_apply(q, pos, r, k=k)[1].sum(), k)  # q's output unused
    check_rope(g, torch.ones((3, 1, 32)), pos.cpu(), inv, layout, factor, -1.0)


def test_rotary_refuses_frequencies_that_want_a_gradient(pkg, cuda_device):
    A, f = pkg.attention, torch.ones(4, device="cuda")
    with pytest.raises(ValueError, match="no gradient"):
        A.Rotary(f.clone().requires_grad_())
    with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError, match="no gradient"):
        A.Rotary(torch.autograd.forward_ad.make_dual(f, f))
    assert A.Rotary(f).rotate_dim == 8


# ---------------------------------------------------------------- the cache


def make_cache(pkg, P, H, blk, D, fmt, junk=True):
    """A cache whose unused memory holds anything (NaN codes for e4m3)."""
    c = pkg.attention.KVCache(P, H, D, blk, fmt)
    if junk:
        for t in (c.k_codes, c.v_codes):
            t.view(torch.uint8).fill_(0x7F)
        c.k_scale.fill_(float("nan"))
        c.v_scale.fill_(float("nan"))
    return c, ref.RefCache(P, H, blk, D, fmt), ref.RefCache(P, H, blk, D, fmt)


def cache_equal(c, rk, rv, pages_lens, blk):
    """Codes and scales of every written token equal the reference's."""
    kc, vc = c.k_codes.cpu().float().double(), c.v_codes.cpu().float().double()
    for pages, n in pages_lens:
        for j in range(-(-n // blk)):
            p, m = int(pages[j]), min(blk, n - j * blk)
            for got, want in ((c.k_scale[p].cpu().double(), rk.scale[p]), (c.v_scale[p].cpu().double(), rv.scale[p])):
                assert torch.equal(torch.isnan(got), torch.isnan(want))
                assert torch.equal(got.nan_to_num(), want.nan_to_num()), (got, want)
            assert torch.equal(kc[p][:, :m], rk.vals[p][:, :m]), (p, (kc[p][:, :m] - rk.vals[p][:, :m]).abs().max())
            assert torch.equal(vc[p][:, :, :m].transpose(1, 2), rv.vals[p][:, :m])


def tables(lens_max, blk, P, seed):
    """Shuffled pages for sequences of up to lens_max tokens; -1 past the end."""
    need = [max(1, -(-n // blk)) for n in lens_max]
    perm = np.random.default_rng(seed).permutation(P)
    t = np.full((len(need), max(need) + 1), -1, np.int64)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = perm[at:at + n]
        at += n
    return t


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,D,blk,layout,rot", [(2, 128, 64, "interleaved", 128), (3, 80, 16, "half", 40), (1, 16, 32, "interleaved", 4),
                                                (2, 256, 64, "half", 256), (2, 48, 16, "interleaved", 0)])
def test_append_and_read(pkg, cuda_device, fmt, dtype, H, D, blk, layout, rot):
    """Four appends (prompts, then a few tokens at a time, growing blocks) into
    ragged sequences: codes and scales after each equal the reference's, as do
    the values read back; q is rotated beside."""
    A = pkg.attention
    steps = [[1, blk + 3, 0, 2 * blk], [1, 1, 1, 1], [3, 0, blk, 5], [1, 1, 1, 0]]
    lens_max = [sum(s[b] for s in steps) for b in range(4)]
    P = sum(-(-n // blk) for n in lens_max) + 2
    c, rk, rv = make_cache(pkg, P, H, blk, D, fmt)
    tab = tables(lens_max, blk, P, 1)
    td = i32(tab.tolist())
    inv = torch.from_numpy((10000.0 ** (-2.0 * np.arange(rot // 2) / max(rot, 1))).astype(np.float32))
    r = A.Rotary(inv.cuda(), layout, 1.0)
    lens = np.zeros(4, int)
    for si, n in enumerate(steps):
        N = sum(n)
        gain = 1.0 + 3.0 * si  # later tokens are larger: scales grow
        k, v = randn((N + 2, H, D), 10 + si, DT[dtype], gain), randn((N + 2, H, D), 20 + si, DT[dtype], gain)
        q = randn((N + 2, 2 * H, D), 30 + si, DT[dtype])
        lens = lens + np.array(n)
        cu = np.concatenate([[0], np.cumsum(n)])
        pos = torch.tensor([p for b in range(4) for p in range(lens[b] - n[b], lens[b])], dtype=torch.int64)
        kr = ref.rotate(k[:N], pos, inv, layout)
        for b in range(4):
            rk.append(kr, int(cu[b]), n[b], int(lens[b]), tab[b])
            rv.append(v[:N].double(), int(cu[b]), n[b], int(lens[b]), tab[b])
        q_out = c.append(k.cuda(), v.cuda(), td, i32(lens.tolist()), cu_of(n), rotary=r, q=q.cuda())
        c.check()
        cache_equal(c, rk, rv, [(tab[b], int(lens[b])) for b in range(4)], blk)
        check_rope(q_out[:N], q[:N], pos, inv, layout, 1.0)
    starts = [0, 2, int(lens[2]), 17]
    counts = [int(lens[b]) - starts[b] for b in range(4)]
    for out in ("bf16", "f32"):
        gk, gv = c.read(td, i32(starts), cu_of(counts), sum(counts), dtype=DT[out], kv_lens=i32(lens.tolist()))
        wk = torch.cat([rk.tokens(tab[b], int(lens[b]))[starts[b]:] for b in range(4)])
        wv = torch.cat([rv.tokens(tab[b], int(lens[b]))[starts[b]:] for b in range(4)])
        assert torch.equal(gk.cpu().double(), wk) and torch.equal(gv.cpu().double(), wv)
    gk, _ = c.read(td[:1], None, i32([0, 2]), 2)
    assert torch.equal(gk.cpu().double(), rk.tokens(tab[0], 2))
    c.check()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,H,D,blk,layout", [("bf16", 11, 128, 64, "half"), ("f32", 22, 64, 16, "interleaved"),
                                                  ("bf16", 6, 256, 32, "interleaved"), ("f32", 10, 144, 64, "half")])
def test_append_long_prompts(pkg, cuda_device, fmt, dtype, H, D, blk, layout):
    """Prompts of more than 1.5 M elements, which keys, values and queries are
    written for in a launch each: a fresh sequence, one that goes on inside a
    block with larger values, an idle one."""
    A = pkg.attention
    P = -(-1200 // blk) + -(-90 // blk) + 1
    c, rk, rv = make_cache(pkg, P, H, blk, D, fmt)
    tab = tables([1200, 90, 0], blk, P, 11)[:, :-(-1200 // blk)]
    inv = torch.from_numpy((10000.0 ** (-2.0 * np.arange(D // 2) / D)).astype(np.float32))
    r = A.Rotary(inv.cuda(), layout, 1.0)
    lens = np.zeros(3, int)
    for si, n in enumerate(([5, 0, 0], [1100, 77, 0], [3, 13, 0])):
        N, cu = sum(n), np.concatenate([[0], np.cumsum(n)])
        k, v = randn((N, H, D), 50 + si, DT[dtype], 1.0 + si), randn((N, H, D), 60 + si, DT[dtype], 1.0 + si)
        q = randn((N, 2 * H, D), 70 + si, DT[dtype])
        lens = lens + np.array(n)
        pos = torch.tensor([p for b in range(3) for p in range(lens[b] - n[b], lens[b])], dtype=torch.int64)
        kr = ref.rotate(k, pos, inv, layout)
        for b in range(3):
            rk.append(kr, int(cu[b]), n[b], int(lens[b]), tab[b])
            rv.append(v.double(), int(cu[b]), n[b], int(lens[b]), tab[b])
        q_out = c.append(k.cuda(), v.cuda(), i32(tab.tolist()), i32(lens.tolist()), cu_of(n), rotary=r, q=q.cuda())
        c.check()
        cache_equal(c, rk, rv, [(tab[b], int(lens[b])) for b in range(3)], blk)
        check_rope(q_out, q, pos, inv, layout, 1.0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rot", [2, 6, 18, 50])
@pytest.mark.parametrize("H,n", [(2, [5, 70, 0]), (17, [900, 600, 1])])
def test_append_half_layout_with_an_odd_half(pkg, cuda_device, fmt, dtype, rot, H, n):
    """rotate_dim / 2 odd in the half layout: the second elements of the pairs
    begin on an odd one, in one launch and in a launch each for q, k and v."""
    A = pkg.attention
    D, blk = 64, 32
    lens_max = [x + 3 for x in n]
    P = sum(-(-x // blk) for x in lens_max)
    c, rk, rv = make_cache(pkg, P, H, blk, D, fmt)
    tab = tables(lens_max, blk, P, 12)
    inv, _ = A.rotary_frequencies(D, 10000.0, (rot + 0.5) / D)
    assert inv.size == rot // 2
    r, inv = A.Rotary(inv, "half"), torch.from_numpy(inv)
    lens = np.zeros(3, int)
    for si, m in enumerate((n, [3, 0, 2])):
        N, cu = sum(m), np.concatenate([[0], np.cumsum(m)])
        k, v = randn((N, H, D), 80 + si, DT[dtype], 1.0 + si), randn((N, H, D), 90 + si, DT[dtype], 1.0 + si)
        q = randn((N, H, D), 95 + si, DT[dtype])
        lens = lens + np.array(m)
        pos = torch.tensor([p for b in range(3) for p in range(lens[b] - m[b], lens[b])], dtype=torch.int64)
        kr = ref.rotate(k, pos, inv, "half")
        for b in range(3):
            rk.append(kr, int(cu[b]), m[b], int(lens[b]), tab[b])
            rv.append(v.double(), int(cu[b]), m[b], int(lens[b]), tab[b])
        q_out = c.append(k.cuda(), v.cuda(), i32(tab.tolist()), i32(lens.tolist()), cu_of(m), rotary=r, q=q.cuda())
        c.check()
        cache_equal(c, rk, rv, [(tab[b], int(lens[b])) for b in range(3)], blk)
        check_rope(q_out, q, pos, inv, "half", 1.0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("held", [0, 3, 21])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_poisoned_block_holds_zero_codes(pkg, cuda_device, fmt, dtype, held, bad):
    """Attention multiplies a masked token's zero weight by its stored code, so a
    poisoned block's codes are zeros: those written with the bad value, the old
    ones before it, and those written after it."""
    D, blk, H = 32, 32, 2
    for which in ("k", "v"):
        c, _, _ = make_cache(pkg, 2, H, blk, D, fmt)
        tab = i32([[1]])
        write = lambda x, end: c.append(*((x, torch.ones_like(x)) if which == "k" else (torch.ones_like(x), x)), tab, i32([end]),
                                        i32([0, x.size(0)]))
        if held:
            write(randn((held, H, D), 120, DT[dtype]).cuda(), held)
        x = randn((4, H, D), 121, DT[dtype])
        x[2, 1, 7] = bad
        write(x.cuda(), held + 4)
        for end in (held + 4, held + 6):
            codes = (c.k_codes[1] if which == "k" else c.v_codes[1].transpose(1, 2)).view(torch.uint8)[:, :end]
            scale = c.k_scale if which == "k" else c.v_scale
            assert torch.isnan(scale[1, 1]) and torch.isfinite(scale[1, 0])
            assert not bool(codes[1].any()) and bool(codes[0].any())
            write(randn((2, H, D), 122, DT[dtype]).cuda(), end + 2)
    c.check()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_grows_a_scale_with_every_token(pkg, cuda_device, fmt):
    """Token after token of twice the size: every write reads the scale that the
    one before left, and rounds all earlier codes again."""
    D, blk, H = 48, 32, 3
    c, rk, rv = make_cache(pkg, 2, H, blk, D, fmt)
    tab = i32([[1, 0]])
    for n in range(1, 41):
        k, v = (randn((1, H, D), 200 * i + n, torch.bfloat16, 2.0 ** (n % 33)) for i in (1, 2))
        rk.append(k.double(), 0, 1, n, [1, 0])
        rv.append(v.double(), 0, 1, n, [1, 0])
        c.append(k.cuda(), v.cuda(), tab, i32([n]), i32([0, 1]))
    cache_equal(c, rk, rv, [([1, 0], 40)], blk)
    c.check()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_values_at_the_edges(pkg, cuda_device, fmt):
    """Zeros, subnormals, values at the scale's border, the largest floats, and
    values that are not finite; a poisoned block reads NaN until it starts over."""
    D, blk, q = 16, 16, ref.QMAX[fmt]
    c, rk, rv = make_cache(pkg, 12, 1, blk, D, fmt)
    rows = [torch.zeros(D), torch.full((D,), 1e-42), torch.full((D,), q), torch.full((D,), q * (1 + 2.0 ** -20)),
            torch.full((D,), 3.4e38), torch.linspace(-q, q, D), torch.full((D,), -2.0 ** -120)]
    tab = i32([[i] for i in range(len(rows))])
    x = torch.stack(rows)[:, None]
    n = len(rows)
    for b in range(n):
        rk.append(x.double(), b, 1, 1, [b])
        rv.append(x.double(), b, 1, 1, [b])
    c.append(x.cuda(), x.cuda(), tab, i32([1] * n), cu_of([1] * n))
    cache_equal(c, rk, rv, [([b], 1) for b in range(n)], blk)
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = torch.ones((3, 1, D))
        y[1, 0, 3] = bad
        t = i32([[9]])
        c.append(y.cuda(), torch.ones_like(y).cuda(), t, i32([3]), i32([0, 3]))
        assert math.isnan(float(c.k_scale[9, 0])) and not math.isnan(float(c.v_scale[9, 0]))
        assert torch.isfinite(c.k_codes[9].float()).all() or fmt == "e4m3"
        c.append(torch.ones((1, 1, D), device="cuda"), torch.ones((1, 1, D), device="cuda"), t, i32([4]), i32([0, 1]))
        gk, gv = c.read(t, None, i32([0, 4]), 4, dtype=torch.float32)
        assert torch.isnan(gk).all() and torch.equal(gv.cpu(), torch.ones((4, 1, D)))
        c.append(torch.ones((1, 1, D), device="cuda"), torch.ones((1, 1, D), device="cuda"), t, i32([1]), i32([0, 1]))
        gk, _ = c.read(t, None, i32([0, 1]), 1, dtype=torch.float32)
        assert torch.equal(gk.cpu(), torch.ones((1, 1, D)))
    c.check()


# ---------------------------------------------------------------- attention


def fill(c, seed, gain=1.0):
    """Random finite codes and power-of-two scales; returns the reference pools."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for codes, scale, trans in ((c.k_codes, c.k_scale, False), (c.v_codes, c.v_scale, True)):
        P, H = scale.shape
        x = torch.randn(codes.shape, generator=g) * (40 if c.format == "int8" else 100)
        x = x.round().clamp(-127, 127).to(torch.int8) if c.format == "int8" else x.clamp(-448, 448).to(ref.F8)
        s = 2.0 ** torch.randint(-8, -4, (P, H), generator=g).float() * gain
        codes.copy_(x.cuda())
        scale.copy_(s.cuda())
        r = ref.RefCache(P, H, c.block, c.head_dim, c.format)
        r.vals = (x.float().double().transpose(2, 3) if trans else x.float().double()).contiguous()
        r.scale = s.double()
        out.append(r)
    return out


def check_attention(pkg, c, rk, rv, tab, lens, news, Hq, dtype, window=0, seed=0, qgain=1.0, scale=None, max_rows=None,
                    strided=False):
    N, D = sum(news), c.head_dim
    q = randn((N, Hq, D), seed, DT[dtype], qgain)
    qd = q.cuda()
    if strided:
        wide = torch.zeros((N, Hq + 3, D), dtype=DT[dtype], device="cuda")
        wide[:, 1:1 + Hq] = qd
        qd = wide[:, 1:1 + Hq]
    pad = 3
    qp = torch.cat([qd, torch.full((pad, Hq, D), float("nan"), dtype=DT[dtype], device="cuda")])
    out = torch.full_like(qp, 7.5)
    got, lse = c.attention(qp, i32(tab.tolist()), i32(lens), cu_of(news), max(news) if max_rows is None else max_rows, scale=scale,
                           window=window, out=out, return_lse=True)
    c.check()
    assert torch.all(got[N:] == 7.5)  # rows behind the last sequence
    row = 0
    sc = scale if scale is not None else D ** -0.5
    for b, (L, n) in enumerate(zip(lens, news)):
        if n == 0:
            continue
        pos = torch.arange(L - n, L)
        o, ls, mag, smax, vsum = ref.attend(q[row:row + n].double(), rk.tokens(tab[b], L), rv.tokens(tab[b], L), pos, sc, window)
        g = got[row:row + n].cpu().double()
        tol = ref.attend_tolerance(DT[dtype], o, mag, smax, vsum, D, L)
        bad = torch.isnan(g) | ((g - o).abs() > tol)
        assert not bool(bad.any()), (b, L, n, float(((g - o).abs() / tol).max()))
        gl = lse[row:row + n].cpu().double()
        lt = 2 * (D + 8) * 2.0 ** -23 * smax + (L + 64) * 2.0 ** -23 + 2.0 ** -22 * ls.abs()
        assert bool(((gl - ls).abs() <= lt)[~torch.isinf(ls)].all()) and torch.equal(torch.isinf(gl), torch.isinf(ls))
        row += n
    return got


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("Hkv,g,D,blk", [(2, 4, 128, 64), (1, 1, 64, 16), (2, 5, 80, 32), (1, 16, 256, 64), (3, 2, 16, 16),
                                         (1, 33, 48, 32), (2, 8, 128, 16), (1, 8, 144, 32)])
def test_attention(pkg, cuda_device, fmt, dtype, Hkv, g, D, blk):
    """Ragged batch: one token, block borders, idle sequences, many rows."""
    lens = [1, blk, blk + 1, 0, 63, 64, 65, 700, 129, 5]
    news = [1, 1, 2, 0, 1, 3, 65, 1, 17, 5]
    P = sum(max(1, -(-n // blk)) for n in lens) + 3
    c, _, _ = make_cache(pkg, P, Hkv, blk, D, fmt)
    rk, rv = fill(c, 5)
    tab = tables(lens, blk, P, 2)
    check_attention(pkg, c, rk, rv, tab, lens, news, Hkv * g, dtype, seed=3)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [1, 16, 63, 64, 200])
def test_attention_window(pkg, cuda_device, dtype, window):
    lens, news, blk = [300, 64, 1, 555, 210], [1, 64, 1, 40, 9], 32
    P = sum(-(-n // blk) for n in lens)
    c, _, _ = make_cache(pkg, P, 2, blk, 64, "int8")
    rk, rv = fill(c, 6)
    check_attention(pkg, c, rk, rv, tables(lens, blk, P, 4), lens, news, 8, dtype, window=window, seed=4, strided=True)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("B,L,Hkv", [(1, 20000, 1), (1, 9000, 8), (300, 90, 2), (3, 4000, 2)])
def test_attention_split(pkg, cuda_device, fmt, B, L, Hkv):
    """Long contexts cut between warps and joined; many short sequences."""
    rng = np.random.default_rng(B)
    lens = [int(x) for x in rng.integers(max(1, L // 2), L + 1, B)]
    blk = 64
    P = sum(-(-n // blk) for n in lens)
    c, _, _ = make_cache(pkg, P, Hkv, blk, 128, fmt)
    rk, rv = fill(c, 7)
    check_attention(pkg, c, rk, rv, tables(lens, blk, P, 5), lens, [1] * B, 4 * Hkv, "bf16", seed=5, qgain=3.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_prompt_from_nothing(pkg, cuda_device, dtype):
    """A whole prompt (its own rows are all the context), with and without a window."""
    lens, blk = [333, 1, 128, 200], 64
    P = sum(-(-n // blk) for n in lens)
    c, _, _ = make_cache(pkg, P, 2, blk, 128, "int8")
    rk, rv = fill(c, 8)
    for w in (0, 50):
        check_attention(pkg, c, rk, rv, tables(lens, blk, P, 6), lens, lens, 8, dtype, window=w, seed=6)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("qgain,gain", [(1e-30, 1.0), (1e30, 2.0 ** -100), (60.0, 1.0), (0.0, 1.0), (1.0, 2.0 ** 60), (1.0, 2.0 ** -60)])
def test_attention_magnitudes(pkg, cuda_device, dtype, qgain, gain):
    """Queries and scales far from one, peaked and flat softmax."""
    lens, blk = [150, 64], 16
    P = 14
    c, _, _ = make_cache(pkg, P, 1, blk, 64, "e4m3")
    rk, rv = fill(c, 9, gain)
    s = 0.125 if gain == 1.0 or qgain != 1.0 else 0.125 / gain
    check_attention(pkg, c, rk, rv, tables(lens, blk, P, 7), lens, [1, 2], 4, dtype, seed=7, qgain=qgain, scale=s)


@pytest.mark.parametrize("D,blk,fmt", [(64, 16, "int8"), (96, 32, "e4m3"), (128, 64, "int8"), (128, 64, "e4m3"), (16, 64, "int8")])
@pytest.mark.parametrize("window", [0, 100])
def test_attention_many_rows(pkg, cuda_device, D, blk, fmt, window):
    """The tensor-core kernel: chunks on cached context, part row tiles, one and
    two row tiles of a block, rows that begin a tile, queries off the vector's
    alignment; sequences with few rows beside them."""
    lens, news = [500, 129, 1, 700, 64, 400], [300, 65, 1, 257, 64, 3]
    P = sum(-(-n // blk) for n in lens) + 1
    c, _, _ = make_cache(pkg, P, 2, blk, D, fmt)
    rk, rv = fill(c, 21)
    tab = tables(lens, blk, P, 8)
    for g in (1, 3, 8):
        check_attention(pkg, c, rk, rv, tab, lens, news, 2 * g, "bf16", window=window, seed=20 + g, strided=g == 3, qgain=2.0)
    N = sum(news)
    q = randn((N, 4, D), 30, torch.bfloat16).cuda()
    flat = torch.empty(N * 4 * D + 1, dtype=torch.bfloat16, device="cuda")
    off = flat[1:].view(N, 4, D)
    off.copy_(q)
    args = (i32(tab.tolist()), i32(lens), cu_of(news), max(news))
    assert torch.equal(c.attention(off, *args, out=torch.empty_like(off)), c.attention(q, *args))
    # a wrong hint costs time, not results: both kernels answer alike but for their sums' order
    a, b = c.attention(q, *args).float(), c.attention(q, *args[:3], 1).float()
    assert float((a - b).abs().max()) <= 2.0 ** -7 * float(b.abs().max())
    assert torch.equal(c.attention(q, *args, scale=-0.07), c.attention(-q, *args, scale=0.07))


@pytest.mark.parametrize("D,blk,fmt", [(64, 64, "int8"), (128, 16, "e4m3"), (80, 32, "int8")])
@pytest.mark.parametrize("lens,news", [([3000], [200]), ([2900, 40, 300], [8, 1, 7]), ([2500, 1, 0, 70], [130, 1, 0, 33]), ([130], [130])])
def test_attention_many_rows_in_parts(pkg, cuda_device, D, blk, fmt, lens, news):
    """Few rows over a long context: the tensor-core kernel cuts the context and
    joins the parts.  Parts without a tile (the table has room for more than the
    sequences hold), windows inside one part and over several, a page that
    cannot be read."""
    P = sum(-(-n // blk) for n in lens) + 1
    c, _, _ = make_cache(pkg, P, 1, blk, D, fmt)
    rk, rv = fill(c, 22)
    tab = tables(lens, blk, P, 9)
    tab = np.concatenate([tab, np.full((len(lens), 3000 // blk), -1, np.int64)], 1)
    for window in (0, 90, 1500):
        check_attention(pkg, c, rk, rv, tab, lens, news, 4, "bf16", window=window, seed=40 + window, qgain=2.0, strided=window == 90)
    q = randn((news[0], 4, D), 41, torch.bfloat16).cuda()
    bad = tab[:1].copy()
    at = (lens[0] - 1) // blk  # the last page: rows before it do not see it
    bad[0, at] = P + 5
    got, lse = c.attention(q, i32(bad.tolist()), i32(lens[:1]), cu_of(news[:1]), news[0], return_lse=True)
    with pytest.raises(RuntimeError, match="page"):
        c.check()
    want = c.attention(q, i32(tab[:1].tolist()), i32(lens[:1]), cu_of(news[:1]), news[0])
    n = max(at * blk - (lens[0] - news[0]), 0)
    assert torch.equal(got[:n], want[:n]) and torch.isnan(got[n:]).all() and torch.isnan(lse[n:]).all()
    c.check()


@pytest.mark.parametrize("lens,news", [([1024], [512]), ([1000, 700], [256, 5]), ([3000, 1, 90], [40, 1, 33]), ([200], [9])])
@pytest.mark.parametrize("window", [0, 300])
def test_a_wider_page_table_changes_nothing(pkg, cuda_device, lens, news, window):
    """How a context is cut goes by the sequences' lengths, not by the room that
    the page table has for more: the answers are the same to the bit."""
    blk, H = 64, 4
    need = [-(-n // blk) for n in lens]
    c, _, _ = make_cache(pkg, sum(need), H, blk, 128, "int8")
    fill(c, 51)
    tab = np.full((len(lens), max(need)), -1, np.int64)
    for b, n in enumerate(need):
        tab[b, :n] = np.arange(n) + sum(need[:b])
    q = randn((sum(news), 4 * H, 128), 52, torch.bfloat16).cuda()
    out = []
    for wide in (0, 8, 2048):
        t = np.concatenate([tab, np.full((len(lens), wide), -1, np.int64)], 1)
        out.append(c.attention(q, i32(t.tolist()), i32(lens), cu_of(news), max(news), window=window, return_lse=True))
    for got, lse in out[1:]:
        assert torch.equal(got, out[0][0]) and torch.equal(lse, out[0][1])
    c.check()


@pytest.mark.parametrize("L", [350, 5000])
def test_overlapping_row_offsets_stay_in_bounds(pkg, cuda_device, L):
    """Offsets that go back: one sequence is skipped, two share rows, and the
    batch has more row tiles than its rows allow."""
    blk, P = 64, -(-5000 // 64)
    c, _, _ = make_cache(pkg, P, 1, blk, 64, "int8")
    fill(c, 24)
    q = torch.cat([randn((300, 4, 64), 43, torch.bfloat16), torch.full((40, 4, 64), 3.0, dtype=torch.bfloat16)]).cuda()
    out = torch.full_like(q, 7.5)
    tab = i32(np.broadcast_to(np.arange(P), (3, P)).tolist())
    got = c.attention(q[:300], tab, i32([L] * 3), i32([0, 300, 100, 300]), 300, out=out[:300])
    with pytest.raises(RuntimeError, match="offsets"):
        c.check()
    assert torch.all(out[300:] == 7.5) and torch.isfinite(got[:100]).all()
    c.read(tab, None, i32([0, 300, 100, 300]), 300)
    with pytest.raises(RuntimeError, match="offsets"):
        c.check()
    want = c.attention(q[:300], tab[:1], i32([L]), i32([0, 300]), 300)  # the cache still answers
    assert torch.isfinite(want).all()
    c.check()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("rows", [16, 128])
@pytest.mark.parametrize("down", [20, 60])
def test_attention_value_scales_far_apart(pkg, cuda_device, fmt, rows, down):
    """Values of the first 128 tokens 2^20 or 2^60 times smaller than the later
    ones: rows that see only the first keep their precision, whether they run
    beside rows that see the others or not."""
    blk, D, L = 32, 64, 700
    P = -(-L // blk)
    c, _, _ = make_cache(pkg, P, 1, blk, D, fmt)
    rk, rv = fill(c, 23)
    tab = tables([L], blk, P, 10)
    first = torch.from_numpy(tab[0, :128 // blk])
    rv.scale[first] *= 2.0 ** -down
    c.v_scale.copy_(rv.scale.float())
    q = randn((L, 2, D), 42, torch.bfloat16)
    got = c.attention(q.cuda(), i32(tab.tolist()), i32([L]), i32([0, L]), L)
    few = torch.cat([c.attention(q[i:i + rows].cuda(), i32(tab.tolist()), i32([i + rows]), i32([0, rows]), rows)
                     for i in range(0, 640, rows)])
    for beg, end in ((0, 128), (128, 640)):
        o, _, mag, smax, vsum = ref.attend(q[beg:end].double(), rk.tokens(tab[0], end), rv.tokens(tab[0], end),
                                           torch.arange(beg, end), D ** -0.5, 0)
        tol = ref.attend_tolerance(torch.bfloat16, o, mag, smax, vsum, D, L)
        for x in (got, few):
            assert bool(((x[beg:end].cpu().double() - o).abs() <= tol).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("D,blk,step", [(64, 16, 80), (128, 32, 96), (96, 64, 64), (144, 16, 48), (256, 64, 128)])
@pytest.mark.parametrize("up", [12, 25, 40, 100])
@pytest.mark.parametrize("window", [0, 20])
def test_hidden_value_scales_leave_a_row_alone(pkg, cuda_device, dtype, fmt, D, blk, step, up, window):
    """Values 2^up larger from token `step` on (with a window: up to there), the
    border inside the kernels' tiles: rows that do not see them keep the bits
    they have without them, beside rows that do, few or many.  f16's floor is
    relative to the largest scale that the row itself sees."""
    L, P = 200, -(-200 // blk)
    c, _, _ = make_cache(pkg, P, 1, blk, D, fmt)
    rk, rv = fill(c, 49)
    big = torch.arange(P) >= step // blk if window == 0 else torch.arange(P) < step // blk
    rv.scale[big] *= 2.0 ** up
    c.v_scale.copy_(rv.scale.float())
    tab, g = i32([list(range(P))]), 4
    k, v = rk.tokens(range(P), L), rv.tokens(range(P), L)
    size = rv.scale[:, 0].repeat_interleave(blk)[:L]  # of each token
    for beg, end in ((0, 200), (step - 5, step + 4), (step + 15, step + 25), (step - 2, step + 7)):
        pos = torch.arange(beg, end)
        q = randn((end - beg, g, D), 50, DT[dtype])
        o, _, mag, smax, _ = ref.attend(q.double(), k[:end], v[:end], pos, D ** -0.5, window)
        sees = (torch.arange(end)[None] <= pos[:, None]) & ((pos[:, None] - torch.arange(end)[None] <= window) | (window == 0))
        most = (sees * size[:end]).amax(-1)
        vsum = (sees.double() @ (v[:end, 0].abs() / size[:end, None]) * most[:, None])[:, None]
        tol = ref.attend_tolerance(DT[dtype], o, mag, smax, vsum, D, end)
        got = c.attention(q.cuda(), tab, i32([end]), i32([0, end - beg]), end - beg, window=window).cpu().double()
        bad = torch.isnan(got) | ((got - o).abs() > tol)
        assert not bool(bad.any()), (beg, end, bad.any(-1).any(-1).nonzero().flatten().tolist())
    c.check()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("down", [10, 16, 20, 24, 26, 28])
@pytest.mark.parametrize("D,blk", [(64, 16), (128, 32)])
def test_values_of_a_small_block_beside_large_ones(pkg, cuda_device, fmt, down, D, blk):
    """All weight on a token whose block's scale is 2^-down of its neighbours', in
    a tile that every row sees whole: its values are off by f16's last place
    relative to the largest scale (2^-25 of it), not more."""
    L, n, P = 240, 100, -(-240 // blk)
    c, _, _ = make_cache(pkg, P, 1, blk, D, fmt)
    rk, rv = fill(c, 53)
    at = blk + 3  # the token, in the second block
    rv.scale[:] = 1.0
    rv.scale[1] = 2.0 ** -down
    c.v_scale.copy_(rv.scale.float())
    key = rk.tokens(range(P), L)[at, 0]
    q = (key * (60.0 / float(key @ key) * D ** 0.5)).expand(n, 4, D).to(torch.bfloat16)  # its score: 60
    tab = i32([list(range(P))])
    got = c.attention(q.cuda(), tab, i32([L]), i32([0, n]), n).cpu().double()
    k, v = rk.tokens(range(P), L), rv.tokens(range(P), L)
    o, _, mag, smax, _ = ref.attend(q.double(), k, v, torch.arange(L - n, L), D ** -0.5, 0)
    vsum = (v[:, 0].abs() / rv.scale[:, 0].repeat_interleave(blk)[:L, None]).sum(0)
    tol = ref.attend_tolerance(torch.bfloat16, o, mag, smax, vsum, D, L) + 2.0 ** -25
    assert bool(((got - o).abs() <= tol).all()), float(((got - o).abs() / tol).max())
    c.check()


@pytest.mark.parametrize("news", [1, 200])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_attention_masked_blocks_may_hold_anything(pkg, cuda_device, news, fmt):
    """A block whose scale is NaN or infinite (or that names no page) spoils the
    rows that see it and no others; memory past the last token is never used."""
    L, blk, D = 640, 64, 64
    c, _, _ = make_cache(pkg, 11, 1, blk, D, fmt)
    rk, rv = fill(c, 31)
    tab = np.arange(10)[None]
    q = randn((news, 4, D), 32, torch.bfloat16).cuda()
    args = (i32([L - 30]), i32([0, news]), news)
    want = {w: c.attention(q, i32(tab.tolist()), *args, window=w) for w in (0, 100)}
    keep = [t.clone() for t in (c.k_scale, c.v_scale)]
    for bad in (float("nan"), float("inf")):
        for which in ("k_scale", "v_scale"):
            getattr(c, which)[1, 0] = bad  # tokens 64 .. 127
            assert torch.isnan(c.attention(q, i32(tab.tolist()), *args)).all()
            got = c.attention(q, i32(tab.tolist()), *args, window=100)
            sees = torch.tensor([(L - 30 - news + i) - 100 <= 127 for i in range(news)])
            assert torch.equal(torch.isnan(got).all(-1).all(-1).cpu(), sees) and torch.equal(torch.isnan(got).any(-1).any(-1).cpu(), sees)
            assert torch.equal(got[~sees], want[100][~sees])
            c.k_scale.copy_(keep[0])
            c.v_scale.copy_(keep[1])
    # the last page past its 34 tokens: junk codes; a later page that no row sees: junk scale
    for t in (c.k_codes.view(torch.uint8)[9, :, 34:], c.v_codes.view(torch.uint8)[9, :, :, 34:]):
        t.fill_(0x7F)
    c.k_scale[10] = c.v_scale[10] = float("nan")
    assert torch.equal(c.attention(q, i32(tab.tolist()), *args), want[0])
    c.check()
    # pages outside the cache
    for page in (-1, 11, 2 ** 31 - 1):
        t = tab.copy()
        t[0, 0] = page
        assert torch.isnan(c.attention(q, i32(t.tolist()), *args)).all()
        with pytest.raises(pkg.api.NoorMoEError):
            c.check()
        got = c.attention(q, i32(t.tolist()), *args, window=100)
        sees = torch.tensor([(L - 30 - news + i) - 100 <= 63 for i in range(news)])
        assert torch.equal(torch.isnan(got).any(-1).any(-1).cpu(), sees) and torch.equal(got[~sees], want[100][~sees])
        k, v = c.read(i32(t.tolist()), None, i32([0, 70]), 70)
        assert torch.isnan(k[:64]).all() and torch.isnan(v[:64]).all() and torch.isfinite(k[64:].float()).all()
        c.status.zero_()
    c.check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("news,blk,window", [(300, 64, 0), (300, 16, 90), (9, 16, 0), (9, 16, 3), (8, 32, 0)])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_scales_that_no_write_leaves_read_as_nan(pkg, cuda_device, dtype, news, blk, window, which):
    """A negative, infinite or too large scale spoils the rows that see its
    block, and no row beside them; reading the block back gives NaN."""
    D, L = 64, 300 if news == 300 else 70
    c, _, _ = make_cache(pkg, 20, 1, blk, D, "int8")
    rk, rv = fill(c, 44)
    at = 64 // blk  # the block of token 64
    q = randn((news, 4, D), 46, DT[dtype])
    args = (i32([list(range(20))]), i32([L]), i32([0, news]), news)
    pos = torch.arange(L - news, L)
    o, _, mag, smax, vsum = ref.attend(q.double(), rk.tokens(range(20), L), rv.tokens(range(20), L), pos, D ** -0.5, window)
    tol = ref.attend_tolerance(DT[dtype], o, mag, smax, vsum, D, L)
    sees = (pos >= 64) & ((pos - window <= 64 + blk - 1) | (window == 0))
    assert bool(sees.any()) and not bool(sees.all())
    scale = getattr(c, which)
    keep = float(scale[at, 0])
    for bad in (-keep, -math.inf, math.inf, 2.0 ** 127, math.nan):
        scale[at, 0] = bad
        got = c.attention(q.cuda(), *args, window=window).cpu().double()
        assert torch.isnan(got[sees]).all(), bad
        assert bool(((got - o).abs() <= tol)[~sees].all()), bad
        gk, gv = c.read(args[0], None, i32([0, 70]), 70, dtype=DT[dtype])
        x, y = (gk, gv) if which == "k_scale" else (gv, gk)
        assert torch.isnan(x[64:64 + blk]).all() and torch.isfinite(x[:64]).all() and torch.isfinite(y).all()
        if blk * at < 70 < blk * (at + 1):  # a write into the block keeps it spoilt
            one = torch.ones((1, 1, D), device="cuda")
            c.append(one, one, args[0], i32([71]), i32([0, 1]))
            assert math.isnan(float(scale[at, 0]))
            c.k_codes.view(torch.uint8).copy_(rk.vals.to(c.k_codes.dtype).cuda().view(torch.uint8))
            c.v_codes.view(torch.uint8).copy_(rv.vals.transpose(2, 3).contiguous().to(c.k_codes.dtype).cuda().view(torch.uint8))
            c.k_scale.copy_(rk.scale.float())
            c.v_scale.copy_(rv.scale.float())
    c.check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("news", [1, 7, 200])
@pytest.mark.parametrize("D,blk", [(64, 16), (128, 64), (144, 32)])
def test_queries_that_are_not_finite(pkg, cuda_device, dtype, news, D, blk):
    """An infinity or a NaN in a query makes its row NaN, whatever the keys (also
    where all scores are minus infinity), and no row beside it."""
    L, P = 260, -(-260 // blk)
    c, _, _ = make_cache(pkg, P, 1, blk, D, "int8")
    fill(c, 47)
    c.k_codes.copy_(torch.where(c.k_codes == 0, torch.ones_like(c.k_codes), c.k_codes))
    c.k_codes[..., 5] = -3  # an infinite query element 5 has scores of minus infinity
    q = randn((news, 4, D), 48, DT[dtype])
    args = (i32([list(range(P))]), i32([L]), i32([0, news]), news)
    want, lse = c.attention(q.cuda(), *args, return_lse=True)
    assert torch.isfinite(want).all() and torch.isfinite(lse).all()
    for bad in (math.inf, -math.inf, math.nan):
        x = q.clone()
        x[news // 2, 1, 5] = bad
        got, gl = c.attention(x.cuda(), *args, return_lse=True)
        hit = torch.zeros((news, 4), dtype=torch.bool, device="cuda")
        hit[news // 2, 1] = True
        assert torch.isnan(got[hit]).all() and torch.isnan(gl[hit]).all(), bad
        assert torch.equal(got[~hit], want[~hit]) and torch.equal(gl[~hit], lse[~hit])
    c.check()


def test_bad_metadata_is_reported_and_touches_nothing(pkg, cuda_device):
    D, blk = 64, 32
    c, _, _ = make_cache(pkg, 6, 1, blk, D, "int8")
    fill(c, 33)
    tab = i32([[0, 1], [2, 3]])
    before = [t.clone() for t in (c.k_codes, c.v_codes, c.k_scale, c.v_scale)]
    x = randn((4, 1, D), 34, torch.bfloat16).cuda()
    for lens, cu in (([65, 2], [0, 2, 4]), ([-1, 2], [0, 2, 2]), ([1, 2], [0, 2, 2]), ([2, 2], [0, 5, 5]), ([2, 2], [3, 1, 1]),
                     ([2, 2], [-2, 0, 0]), ([2 ** 31 - 1, 2], [0, 2, 2])):
        out = torch.full_like(x, 3.0)
        c.attention(x, tab, i32(lens), i32(cu), 4, out=out)
        with pytest.raises(pkg.api.NoorMoEError):
            c.check()
        if lens[0] != 1:  # (rows at positions below 0 see nothing)
            assert torch.all(out[:2] == 3.0)
        c.append(x, x, i32([[0, 1], [2, 3]]), i32(lens), i32([min(max(v, -5), 9) for v in cu]))
        torch.cuda.synchronize()
        # sequence 1 is sound in the first case alone
        pages = [0, 1, 4, 5] if lens[0] == 65 else range(6)
        for t, b in zip((c.k_codes, c.v_codes, c.k_scale, c.v_scale), before):
            assert torch.equal(t.view(torch.int8)[list(pages)] if t.dtype == torch.int8 else t[list(pages)], b[list(pages)])
        with pytest.raises(pkg.api.NoorMoEError):
            c.check()
        for t, b in zip((c.k_codes, c.v_codes, c.k_scale, c.v_scale), before):
            t.copy_(b)
    c.read(tab, i32([60, 0]), i32([0, 8, 9]), 9)  # past the pages
    with pytest.raises(pkg.api.NoorMoEError):
        c.check()
    c.append(x, x, i32([[6, -1], [2, 3]]), i32([2, 2]), i32([0, 2, 4]))
    with pytest.raises(pkg.api.NoorMoEError):
        c.check()
    assert torch.equal(c.k_codes[:2], before[0][:2])
    c.check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,L", [(3, 2), (3, 0), (90, 89), (300, 40)])
@pytest.mark.parametrize("window", [0, 5])
def test_attention_skips_a_sequence_shorter_than_its_rows(pkg, cuda_device, dtype, n, L, window):
    """Rows that would lie before the sequence's first token: the sequence is
    skipped and reported, its rows stay as they were, the others are answered."""
    blk, D = 32, 64
    c, _, _ = make_cache(pkg, 24, 1, blk, D, "int8")
    fill(c, 38)
    tab = i32(np.arange(24).reshape(2, 12).tolist())
    q = randn((n + 7, 4, D), 39, DT[dtype]).cuda()
    out = torch.full_like(q, 7.5)
    c.attention(q, tab, i32([L, 200]), i32([0, n, n + 7]), n, window=window, out=out)
    with pytest.raises(pkg.api.NoorMoEError, match="length"):
        c.check()
    assert torch.all(out[:n] == 7.5)
    want = c.attention(q[n:], tab[1:], i32([200]), i32([0, 7]), n, window=window)
    # the other's context is cut elsewhere beside it: f32 sums in another order, then one rounding
    assert float((out[n:].float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max())
    c.check()


def test_check_waits_for_other_streams(pkg, cuda_device):
    """A mistake found by a call that is still queued on another stream is not
    missed."""
    c, _, _ = make_cache(pkg, 4, 1, 16, 16, "int8", junk=False)
    x = torch.ones((1, 1, 16), device="cuda")
    tab, lens, cu = i32([[4]]), i32([1]), i32([0, 1])  # page 4 of 4
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c.append(x, x, i32([[0]]), lens, cu)
    c.check()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # a tenth of a second of work ahead of it
        c.append(x, x, tab, lens, cu)
    with pytest.raises(pkg.api.NoorMoEError, match="page"):
        c.check()
    c.check()


def test_attention_in_place_and_shared_pages(pkg, cuda_device):
    """out may be q; sequences may share pages (a common prefix)."""
    blk, D = 16, 48
    c, _, _ = make_cache(pkg, 8, 2, blk, D, "e4m3")
    rk, rv = fill(c, 35)
    tab = np.array([[3, 5, 0, 1], [3, 5, 2, 6], [3, 3, 3, 3]])
    lens, news = [50, 61, 64], [1, 40, 2]
    for dt in ("bf16", "f32"):
        check_attention(pkg, c, rk, rv, tab, lens, news, 6, dt, seed=36)
        q = randn((43, 6, D), 37, DT[dt]).cuda()
        args = (i32(tab.tolist()), i32(lens), cu_of(news), 40)
        want = c.attention(q, *args)
        assert c.attention(q, *args, out=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_offsets_past_32_bits(pkg, cuda_device, fmt):
    """Pages whose byte offsets pass 2^32 are written, read and attended to."""
    P, H, blk, D = 33000, 8, 64, 256  # 4.3 GB a pool
    c, rk_, rv_ = make_cache(pkg, P, H, blk, D, fmt, junk=False)
    pages = [P - 1, 5, P - 2]
    tab = i32([pages])
    n = 130
    k, v = randn((n, H, D), 41, torch.bfloat16), randn((n, H, D), 42, torch.bfloat16)
    rk, rv = (ref.RefCache(3, H, blk, D, fmt) for _ in range(2))
    rk.append(k.double(), 0, n, n, [0, 1, 2])
    rv.append(v.double(), 0, n, n, [0, 1, 2])
    c.append(k.cuda(), v.cuda(), tab, i32([n]), i32([0, n]))
    gk, gv = c.read(tab, None, i32([0, n]), n)
    assert torch.equal(gk.cpu().double(), rk.tokens([0, 1, 2], n)) and torch.equal(gv.cpu().double(), rv.tokens([0, 1, 2], n))
    q = randn((3, 16, D), 43, torch.bfloat16)
    got = c.attention(q.cuda(), tab, i32([n]), i32([0, 3]), 3).cpu().double()
    o, _, mag, smax, vsum = ref.attend(q.double(), rk.tokens([0, 1, 2], n), rv.tokens([0, 1, 2], n), torch.arange(n - 3, n), D ** -0.5, 0)
    assert bool(((got - o).abs() <= ref.attend_tolerance(torch.bfloat16, o, mag, smax, vsum, D, n)).all())
    c.check()


def test_graphs_and_streams(pkg, cuda_device):
    """One captured decode step replays over growing lengths; two graphs and two
    streams do not disturb one another; calls run on the current stream."""
    A = pkg.attention
    D, blk, H, Hq, B = 64, 16, 2, 4, 3
    r = A.Rotary.create(D, device=0)

    class Side:
        def __init__(self, seed):
            self.c, _, _ = make_cache(pkg, 24, H, blk, D, "e4m3")
            self.tab = i32(np.arange(24).reshape(3, 8).tolist())
            self.lens = torch.zeros(B, dtype=torch.int32, device="cuda")
            self.cu = i32([0, 1, 2, 3])
            g = torch.Generator(device="cuda").manual_seed(seed)
            self.xs = [[torch.randn((B, h, D), device="cuda", generator=g).bfloat16() for h in (Hq, H, H)] for _ in range(40)]
            self.q, self.k, self.v = (t.clone() for t in self.xs[0])

        def step(self):
            self.lens += 1
            q = self.c.append(self.k, self.v, self.tab, self.lens, self.cu, rotary=r, q=self.q)
            return self.c.attention(q, self.tab, self.lens, self.cu, 1)

        def eager(self):
            outs = []
            for x in self.xs:
                for d, s in zip((self.q, self.k, self.v), x):
                    d.copy_(s)
                outs.append(self.step().clone())
            return outs

    want = [Side(s).eager() for s in (1, 2)]
    sides = [Side(1), Side(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for s, st in zip(sides, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            s.step()
            s.lens.zero_()
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(s.step())
        s.lens.zero_()
        graphs.append(g)
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(40):
        for j, (s, st, g) in enumerate(zip(sides, streams, graphs)):  # both at once, each on its stream
            with torch.cuda.stream(st):
                for d, x in zip((s.q, s.k, s.v), s.xs[i]):
                    d.copy_(x)
                g.replay()
                got[j].append(outs[j].clone())
    torch.cuda.synchronize()
    for j in range(2):
        sides[j].c.check()
        for i in range(40):
            assert torch.equal(got[j][i], want[j][i]), (j, i)


def test_rope_gradient_in_a_graph_and_twice(pkg, cuda_device):
    """Forward and backward captured together; the gradient's own gradient."""
    A = pkg.attention
    r = A.Rotary.create(32, device=0, layout="half")
    pos = i32([3, 9, 1])
    w = randn((3, 2, 32), 51).cuda()
    x = randn((3, 2, 32), 52).cuda().requires_grad_()
    (want,) = torch.autograd.grad((A.rope_apply(x, pos, r) * w).sum(), x)
    y = randn((3, 2, 32), 52).cuda().requires_grad_()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        torch.autograd.grad((A.rope_apply(y, pos, r) * w).sum(), y)
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        (got,) = torch.autograd.grad((A.rope_apply(y, pos, r) * w).sum(), y)
    got.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    # d/dx of sum(R^T(w x) v): R^T differentiates to R again
    v = randn((3, 2, 32), 53).cuda()
    z = randn((3, 2, 32), 54).cuda().requires_grad_()
    (g1,) = torch.autograd.grad((A.rope_apply(z, pos, r) ** 2).sum(), z, create_graph=True)
    (g2,) = torch.autograd.grad((g1 * v).sum(), z)
    assert float((g2 - 2 * v).abs().max()) <= 1e-5  # R^T R = 1


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_forward_derivative(pkg, cuda_device, dtype, layout):
    """Rotation is linear: a tangent comes out rotated as its input is, for q, k
    or both, also through its gradient and where gradients are off."""
    A, fw = pkg.attention, torch.autograd.forward_ad
    inv, factor = A.rotary_frequencies(32, 10000.0, 0.75, yarn={"scale": 4.0, "original": 2048})
    r, inv = A.Rotary(inv, layout, factor), torch.from_numpy(inv)
    pos = i32([5, 0, 4096])
    q, k, tq, tk = (randn((3, h, 32), 110 + i, DT[dtype]) for i, h in enumerate((2, 1, 2, 1)))
    with fw.dual_level():
        dq, dk = fw.make_dual(q.cuda(), tq.cuda()), fw.make_dual(k.cuda(), tk.cuda())
        for gq, gk, with_grad in ((dq, dk, True), (dq, k.cuda(), True), (q.cuda(), dk, False), (dq, None, False)):
            with torch.set_grad_enabled(with_grad):
                out = A.rope_apply(gq, pos, r, k=gk)
            out = out if gk is not None else (out,)
            for o, x, t, dual in zip(out, (q, k), (tq, tk), (gq is dq, gk is dk)):
                p, tangent = fw.unpack_dual(o)
                check_rope(p, x, pos.cpu(), inv, layout, factor)
                if dual:
                    check_rope(tangent, t, pos.cpu(), inv, layout, factor)
                else:
                    assert tangent is None or not bool(tangent.any())
        # the tangent of the gradient of sum(w . rope(q) . rope(q)) along tq is R^T(w . 2 R tq)
        x = fw.make_dual(q.cuda().float().requires_grad_(), tq.cuda().float())
        y = A.rope_apply(x, pos, r)
        (g,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
        tangent = fw.unpack_dual(g).tangent
        want = ref.rotate(2 * ref.rotate(tq, pos.cpu(), inv, layout, factor), pos.cpu(), inv, layout, factor, -1.0)
        assert float((tangent.detach().cpu().double() - want).abs().max()) <= 64 * 2.0 ** -24 * 2 * factor ** 2 * 6
        c = A.KVCache(2, 1, 32)
        args = (i32([[0, 1]]), i32([3]), i32([0, 3]))
        x = k.cuda()
        for call in (lambda: c.append(dk, x, *args), lambda: c.append(x, dk, *args), lambda: c.append(x, x, *args, rotary=r, q=dq),
                     lambda: c.attention(dq, *args, 3)):
            for with_grad in (True, False):
                with torch.set_grad_enabled(with_grad), pytest.raises(ValueError, match="tangents"):
                    call()
    c.check()


def test_stack_served_from_the_cache(pkg, cuda_device):
    """NoorStack.forward_cached: the attention half against its plain form (the
    projections, the cache and the attention of one layer), and a prompt at once
    against the same tokens a few at a time.  e4m3 blocks grow without loss but
    for codes under 2^-6 of a step's scale (2^-19 of the block's largest
    value), so both ways agree to f32's sums: 1e-4."""
    api, S = pkg.api, pkg.stack
    rng = np.random.default_rng(5)
    att = S.GQAAttention(64, 4, 2, 32, 24, 0.3, rng)
    rope = S.RoPE(32, 10000.0)
    x = randn((50, 64), 61)

    class One:
        blocks, device = [type("B", (), {"attention": att})], 0

    cache = S.StackCache(One, 1, 96, block=16, fmt="int8")
    rows = cache.step([50])
    got = att.forward_cached(x.cuda(), rope, cache.layers[0], rows).cpu().double()
    w = {n: torch.from_numpy(getattr(att, n)).double() for n in ("wq", "wk", "wv", "wo")}
    q, k, v = ((x.double() @ w[n]).view(50, -1, 32) for n in ("wq", "wk", "wv"))
    pos, inv = torch.arange(50), torch.from_numpy(rope.inv_freq)
    rk, rv = ref.RefCache(6, 2, 16, 32, "int8"), ref.RefCache(6, 2, 16, 32, "int8")
    rk.append(ref.rotate(k, pos, inv, "interleaved"), 0, 50, 50, range(6))
    rv.append(v, 0, 50, 50, range(6))
    o, _, mag, smax, vsum = ref.attend(ref.rotate(q, pos, inv, "interleaved"), rk.tokens(range(6), 50), rv.tokens(range(6), 50), pos,
                                 32 ** -0.5, 24)
    want = o.reshape(50, -1) @ w["wo"]
    # a projection off by 2^-20 may round a code the other way: one step of its
    # block for such a token, in k (through the score) and v
    step = float(torch.maximum(rk.scale.max(), rv.scale.max()))
    tol = (ref.attend_tolerance(torch.float32, o, mag, smax, vsum, 32, 50) + 2.0 ** -14 * mag).reshape(50, -1) @ w["wo"].abs() + 1e-5
    bad = (got - want).abs() > tol
    assert float(bad.double().mean()) <= 0.02 and float((got - want).abs().max()) <= 4 * step, (float(bad.double().mean()), step)

    st = S.NoorStack(vocab_size=61, d_model=64, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=32, dense_ffn_dim=128,
                     expert_ffn_dim=64, n_experts=4, n_active_experts=2, sliding_window=8, global_every_n=2, prope_fraction=0.25,
                     dtype=api.DTYPE_F32, rng=rng)
    ids = [list(rng.integers(0, 61, 37)), list(rng.integers(0, 61, 20))]
    c1 = st.new_cache(2, 64, block=16, fmt="e4m3")
    full, util = st.forward_cached(ids, c1)
    c1.check()
    assert full.shape == (57, 61) and torch.isfinite(full).all() and len(util) == 2
    c2 = st.new_cache(2, 64, block=16, fmt="e4m3")
    last = {}
    at = [0, 0]
    for n in ([30, 1], [1, 0], [0, 12], [5, 1], [1, 6]):
        out, _ = st.forward_cached([ids[b][at[b]:at[b] + n[b]] for b in range(2)], c2)
        rows = [0, n[0], n[0] + n[1]]
        for b in range(2):
            at[b] += n[b]
            if n[b]:
                last[b] = out[rows[b + 1] - 1]
    assert at == [37, 20]
    for b, row in ((0, 36), (1, 56)):
        assert float((last[b] - full[row]).norm() / full[row].norm()) <= 1e-4
    with pytest.raises(ValueError):
        st.forward_cached([[1] * 30, []], c2)  # past max_tokens
    with pytest.raises(ValueError):
        st.forward_cached([[99], [1]], c2)
    c2.reset(0)
    again, _ = st.forward_cached([ids[0], []], c2)
    assert float((again[-1] - full[36]).norm() / full[36].norm()) <= 1e-4
    for b in st.blocks:
        b.parallel_ffn.moe.invalidate()


def test_stack_step_that_fails_is_not_counted(pkg, cuda_device):
    """A layer that raises in the middle of a step: the cache holds what it held,
    and the same tokens again give what they would have given."""
    S = pkg.stack
    rng = np.random.default_rng(6)
    st = S.NoorStack(vocab_size=31, d_model=64, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=32, dense_ffn_dim=128,
                     expert_ffn_dim=64, n_experts=4, n_active_experts=2, sliding_window=8, global_every_n=2, prope_fraction=0.25,
                     dtype=pkg.api.DTYPE_F32, rng=rng)
    ids = [list(rng.integers(0, 31, 20)), list(rng.integers(0, 31, 9))]
    clean, broken = st.new_cache(2, 32, block=16), st.new_cache(2, 32, block=16)
    for c in (clean, broken):
        st.forward_cached([ids[0][:12], ids[1][:8]], c)
    want, _ = st.forward_cached([ids[0][12:], ids[1][8:]], clean)
    block, fine = st.blocks[1], st.blocks[1].forward_cached

    def fails(*a):
        raise RuntimeError("planted")

    block.forward_cached = fails
    with pytest.raises(RuntimeError, match="planted"):
        st.forward_cached([ids[0][12:], ids[1][8:]], broken)
    block.forward_cached = fine
    assert broken.lens == [12, 8]
    got, _ = st.forward_cached([ids[0][12:], ids[1][8:]], broken)
    assert broken.lens == [20, 9] and float((got - want).norm() / want.norm()) <= 1e-4
    broken.check()
    for b in st.blocks:
        b.parallel_ffn.moe.invalidate()


def test_cached_path_refuses_gradients_and_takes_any_window(pkg, cuda_device):
    c = pkg.attention.KVCache(4, 1, 16, 16)
    x = torch.ones((1, 1, 16), device="cuda", requires_grad=True)
    args = (i32([[2, 1, -1, -1]]), i32([20]), i32([0, 1]))
    for call in (lambda: c.append(x, x.detach(), *args), lambda: c.append(x.detach(), x, *args), lambda: c.attention(x, *args, 1)):
        with pytest.raises(ValueError, match="no gradient"):
            call()
    rk, rv = fill(c, 30)
    want = c.attention(x.detach(), *args, 1)
    with torch.no_grad():
        for window in (20, 2 ** 31 - 1, 2 ** 31, 2 ** 40 + 5):
            assert torch.equal(c.attention(x, *args, 1, window=window), want)
        rows = torch.ones((20, 1, 16), device="cuda", dtype=torch.bfloat16)
        many = c.attention(rows.repeat(1, 8, 1), args[0], args[1], i32([0, 20]), 20)
        assert torch.equal(c.attention(rows.repeat(1, 8, 1), args[0], args[1], i32([0, 20]), 20, window=2 ** 31 - 1), many)
    c.check()


def test_one_graph_serves_changing_prompts(pkg, cuda_device):
    """The kernels cut contexts by what the device metadata says at replay: one
    captured call over prompts, single rows and idle sequences as they change,
    beside the same call on another stream."""
    blk, P = 32, 3 * (2000 // 32 + 1)
    c, _, _ = make_cache(pkg, P, 1, blk, 64, "int8")
    fill(c, 26)
    tab = i32(np.arange(P).reshape(3, -1).tolist())
    q = randn((216, 4, 64), 45, torch.bfloat16).cuda()
    lens, cu = i32([2000, 300, 5]), i32([0, 200, 215, 216])
    out = torch.empty_like(q)
    call = lambda out=None: c.attention(q, tab, lens, cu, 216, out=out)
    call(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    side = torch.cuda.Stream()
    for new_lens, new_cu in (([2000, 300, 5], [0, 200, 215, 216]), ([216, 2000, 2000], [0, 216, 216, 216]),
                             ([2000, 1999, 1], [0, 1, 2, 3]), ([700, 2000, 40], [0, 8, 176, 216])):
        lens.copy_(i32(new_lens))
        cu.copy_(i32(new_cu))
        out.fill_(7.5)
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            other = call()
        torch.cuda.current_stream().wait_stream(side)
        other.record_stream(torch.cuda.current_stream())
        n = new_cu[-1]
        assert torch.equal(out[:n], other[:n]) and torch.all(out[n:] == 7.5) and torch.isfinite(out).all()
        assert torch.equal(call()[:n], out[:n])
    c.check()
