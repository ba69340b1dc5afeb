"""CPU: what the attention half's entry points refuse (before any CUDA call,
so the pointers here are never used), the Python layer's refusals, and the
rotary tables."""
import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

P = 1 << 20  # a pointer that is aligned and never read
INVALID, UNSUPPORTED = 1, 7
NO_DEVICE = 1 << 20  # a device number that is refused before any launch


def _cache(api, **kw):
    d = dict(k_codes=P, v_codes=P, k_scale=P, v_scale=P, status=0, num_blocks=8, n_kv_heads=2, head_dim=64, block=64,
             format=0, device=0)
    d.update(kw)
    return api.KVCacheDesc(*d.values())


def _batch(api, **kw):
    d = dict(block_table=P, table_stride=4, kv_lens=P, cu_rows=P, n_rows=4, batch=2, max_blocks=4)
    d.update(kw)
    return api.KVBatch(*d.values())


def _heads(api, data=P):
    return api.Heads(data, 128, 64)


def _call(api, name, **kw):
    """One entry point with good arguments but for those given; None passes null."""
    r = ctypes.byref
    opt = lambda v: r(v) if v is not None else None
    g = lambda k, d: kw.get(k, d)
    c, b = g("cache", _cache(api)), g("batch", _batch(api))
    q, out, k, v = g("q", _heads(api)), g("out", _heads(api)), g("k", _heads(api)), g("v", _heads(api))
    rot, dt = g("rotary", api.RotaryDesc(P, 64, 0, 1.0)), g("dtype", 1)
    L = api.lib()
    if name == "rope":
        return L.noor_rope_apply(opt(rot), opt(q), opt(out), g("q_heads", 4), opt(g("rk", None)), opt(g("rk_out", None)),
                                 g("k_heads", 0), g("positions", P), g("tokens", 3), g("head_dim", 64), dt, 0,
                                 g("device", 0), None)
    if name == "append":
        return L.noor_kv_append(opt(c), opt(b), opt(k), opt(v), opt(rot), opt(q), opt(out), g("q_heads", 4), dt, None)
    if name == "read":
        return L.noor_kv_read(opt(c), opt(b), None, g("k_out", P), g("v_out", P), dt, None)
    return L.noor_kv_attention(opt(c), opt(b), opt(q), opt(out), None, g("q_heads", 4), g("max_rows", 1), g("scale", 0.1),
                               g("window", 0), dt, g("workspace", P), g("bytes", 1 << 30), None)


CACHE = [(dict(k_codes=0), INVALID), (dict(v_scale=0), INVALID), (dict(v_codes=P + 8), INVALID), (dict(block=48), UNSUPPORTED),
         (dict(block=128), UNSUPPORTED), (dict(head_dim=24), UNSUPPORTED), (dict(head_dim=272), UNSUPPORTED),
         (dict(head_dim=0), UNSUPPORTED), (dict(format=2), INVALID), (dict(num_blocks=0), INVALID),
         (dict(num_blocks=1 << 33), INVALID), (dict(n_kv_heads=0), INVALID), (dict(device=-1), INVALID)]
BATCH = [(dict(block_table=0), INVALID), (dict(cu_rows=0), INVALID), (dict(batch=0), INVALID), (dict(n_rows=-1), INVALID),
         (dict(n_rows=1 << 30), INVALID), (dict(max_blocks=0), INVALID), (dict(max_blocks=1 << 26), INVALID),
         (dict(table_stride=-1), INVALID)]


@pytest.mark.parametrize("name", ["append", "read", "attention"])
def test_cache_and_batch_refusals(pkg, name):
    api = pkg.api
    for kw, code in CACHE:
        assert _call(api, name, cache=_cache(api, **kw)) == code, kw
        assert api.lib().noor_moe_last_error()
    for kw, code in BATCH:
        assert _call(api, name, batch=_batch(api, **kw)) == code, kw
    if name != "read":
        assert _call(api, name, batch=_batch(api, kv_lens=0)) == INVALID
    assert _call(api, name, cache=None) == INVALID and _call(api, name, batch=None) == INVALID
    assert _call(api, name, dtype=2) == INVALID


def test_call_refusals(pkg):
    api = pkg.api
    odd = _heads(api, P + 1)
    for kw in (dict(k=None), dict(v=_heads(api, 0)), dict(k=odd), dict(out=None), dict(q_heads=0),
               dict(rotary=api.RotaryDesc(0, 64, 0, 1.0)), dict(rotary=api.RotaryDesc(P, 66, 0, 1.0)),
               dict(rotary=api.RotaryDesc(P, 7, 0, 1.0)), dict(rotary=api.RotaryDesc(P, 64, 2, 1.0))):
        assert _call(api, "append", **kw) == INVALID, kw
    for kw in (dict(k_out=0), dict(v_out=P + 8)):
        assert _call(api, "read", **kw) == INVALID, kw
    for kw in (dict(q=None), dict(out=_heads(api, 0)), dict(q_heads=3), dict(q_heads=0), dict(max_rows=-1), dict(window=-1),
               dict(scale=math.inf), dict(scale=math.nan), dict(workspace=0), dict(workspace=P + 4)):
        assert _call(api, "attention", **kw) == INVALID, kw
    for kw, code in ((dict(rotary=None), INVALID), (dict(head_dim=63), UNSUPPORTED), (dict(head_dim=1026), UNSUPPORTED),
                     (dict(head_dim=32), INVALID), (dict(tokens=-1), INVALID), (dict(q_heads=0), INVALID), (dict(q=None), INVALID),
                     (dict(q=odd), INVALID), (dict(positions=0), INVALID), (dict(rk=_heads(api), rk_out=None, k_heads=1), INVALID),
                     (dict(rk=_heads(api), rk_out=_heads(api), k_heads=0), INVALID)):
        assert _call(api, "rope", **kw) == code, kw
    # nothing to do is not an error, and needs no device
    empty = _batch(api, n_rows=0)
    assert _call(api, "rope", tokens=0) == 0
    assert all(_call(api, n, batch=empty) == 0 for n in ("append", "read", "attention"))
    assert api.lib().noor_kv_attention_workspace(ctypes.byref(_cache(api)), ctypes.byref(_batch(api)), 4, 1, 1, None) == INVALID


def test_outputs_whose_heads_overlap_are_refused(pkg):
    api = pkg.api
    for st, sh in ((0, 64), (256, 0), (63, 64), (256, 63), (256, -8)):
        o = api.Heads(P, st, sh)
        assert _call(api, "attention", out=o) == INVALID and _call(api, "append", out=o) == INVALID
        assert _call(api, "rope", out=o) == INVALID and _call(api, "rope", rk=_heads(api), rk_out=o, k_heads=2) == INVALID
        assert b"overlap" in api.lib().noor_moe_last_error()
    # accepted (up to the device, which no machine has): one token and one head, whose strides are not used
    one = api.Heads(P, 0, 0)
    assert _call(api, "rope", out=one, tokens=1, q_heads=1, device=NO_DEVICE) != 0
    assert b"overlap" not in api.lib().noor_moe_last_error()
    assert _call(api, "attention", out=api.Heads(P, 64, 10 ** 6), cache=_cache(api, device=NO_DEVICE)) != 0
    assert b"overlap" not in api.lib().noor_moe_last_error()


def test_rows_past_32_bits_are_refused(pkg):
    """Row and query head of a group are numbered in 32 bits."""
    api = pkg.api
    n = ctypes.c_int64()

    def need(rows, q_heads, kv_heads):
        return api.lib().noor_kv_attention_workspace(ctypes.byref(_cache(api, n_kv_heads=kv_heads)),
                                                     ctypes.byref(_batch(api, n_rows=rows)), q_heads, 1, 1, ctypes.byref(n))

    assert need(1 << 28, 8, 1) == INVALID and need((1 << 25) - 4, 64, 1) == INVALID
    # (the answer itself needs a device)
    assert need(1 << 28, 14, 2) != INVALID and need((1 << 25) - 5, 64, 1) != INVALID
    for rows, heads in ((1 << 28, 16), (1 << 26, 64)):
        assert _call(api, "attention", cache=_cache(api, n_kv_heads=1), batch=_batch(api, n_rows=rows), q_heads=heads,
                     bytes=1 << 62) == INVALID
        assert b"32 bits" in api.lib().noor_moe_last_error()


@pytest.mark.parametrize("name", ["append", "read"])
def test_blocks_past_32_bits_are_refused(pkg, name):
    """256 sequences that (by overlapping offsets) have all the rows each touch
    fewer than 2^31 blocks."""
    api = pkg.api
    for rows, block, ok in ((1 << 28, 16, False), (1 << 28, 32, False), (1 << 28, 64, True), (1 << 26, 16, True)):
        # (accepted up to the device, which no machine has)
        assert _call(api, name, cache=_cache(api, block=block, device=NO_DEVICE), batch=_batch(api, n_rows=rows)) != 0
        assert (b"n_rows" in api.lib().noor_moe_last_error()) != ok, (rows, block)


def test_python_refuses_cpu_tensors(pkg):
    A = pkg.attention
    with pytest.raises(ValueError):
        A.Rotary(torch.ones(4))
    with pytest.raises(ValueError):
        A.rope_apply(torch.ones(2, 2, 8), torch.zeros(2, dtype=torch.int32), None)
    with pytest.raises(ValueError):
        A.KVCache.from_tensors(torch.zeros(2, 2, 64, 16, dtype=torch.int8), torch.zeros(2, 2, 16, 64, dtype=torch.int8),
                               torch.zeros(2, 2), torch.zeros(2, 2))
    with pytest.raises(ValueError):
        A.KVCache(4, 2, 64, fmt="int4")


def test_rotary_tables(pkg):
    """The reference's frequencies, and the stretched ones at their fixed points."""
    A, S = pkg.attention, pkg.stack
    for D, th, fr in ((64, 10000.0, None), (128, 1e6, 0.25), (80, 1e4, 0.3)):
        inv, f = A.rotary_frequencies(D, th, fr)
        want, rot = S.rope_inv_freq(D, th, fr)
        assert f == 1.0 and inv.size == rot // 2
        np.testing.assert_allclose(inv, want, rtol=2.0 ** -23)
    base, _ = A.rotary_frequencies(128)
    lin, _ = A.rotary_frequencies(128, linear=4.0)
    np.testing.assert_allclose(lin, base / 4, rtol=2.0 ** -22)
    ntk, _ = A.rotary_frequencies(128, ntk=4.0)
    np.testing.assert_allclose([ntk[0], ntk[-1]], [base[0], base[-1] / 4], rtol=1e-5)  # fastest kept, slowest stretched
    yarn, f = A.rotary_frequencies(128, yarn={"scale": 8.0, "original": 4096})
    turns = 4096 * base.astype(np.float64) / (2 * math.pi)
    np.testing.assert_allclose(yarn[turns > 33], base[turns > 33], rtol=1e-6)
    np.testing.assert_allclose(yarn[turns < 0.99], base[turns < 0.99] / 8, rtol=1e-6)
    assert np.all(yarn <= base * (1 + 1e-6)) and np.all(yarn >= base / 8 * (1 - 1e-6)) and abs(f - (0.1 * math.log(8) + 1)) < 1e-12
    for bad in (dict(linear=2.0, ntk=2.0), dict(linear=0.0), dict(yarn={"scale": -1.0, "original": 8})):
        with pytest.raises(ValueError):
            A.rotary_frequencies(64, **bad)


@pytest.mark.parametrize("bad", [dict(theta=0.0), dict(theta=math.nan), dict(theta=-1e4), dict(linear=math.inf), dict(linear=math.nan),
                                 dict(ntk=math.nan), dict(yarn={"scale": math.nan, "original": 8}),
                                 dict(yarn={"scale": 2.0, "original": 0}), dict(yarn={"scale": 2.0, "original": 8, "fast": 1.0}),
                                 dict(yarn={"scale": 2.0, "original": 8, "slow": 40.0}),
                                 dict(yarn={"scale": 2.0, "original": 8, "slow": math.nan})])
def test_rotary_tables_refuse_what_gives_no_frequencies(pkg, bad):
    with pytest.raises(ValueError):
        pkg.attention.rotary_frequencies(64, **bad)


# ---- what no run can show: rules of the memory model and of warp votes, read from the sources


def _source(name):
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "noor_-_bangla_ai_b200", "csrc", name)) as f:
        return f.read()


def test_streamed_wait_votes_with_all_its_lanes():
    """A barrier's test may answer the lanes of a warp differently, so no lane
    leaves the wait before the warp's vote."""
    s = _source("kv_attention.cuh")
    body = s[s.index("auto wait = [&]"):]
    body = body[:body.index("    };")]
    assert "mbar_try_wait" in body and "return" not in body
    assert body.rstrip().splitlines()[-1].strip().startswith("if (__any_sync(0xffffffffu")


def test_what_a_running_grid_writes_is_not_loaded_as_read_only():
    """The read-only path wants data that no resident grid writes: the join waits
    for a grid that writes its parts' list, and the write replaces the scales
    that it reads."""
    join = _source("kv_attention.cuh")
    join = join[join.index("combine_kernel(const Args a) {"):]
    assert "a.desc" in join and not [w for w in ("desc", "part_ml", "part_o") if f"__ldg(a.{w}" in join]
    write = _source("kv_cache.cuh")
    write = write[write.index("void append_keys"):write.index("// Rotate q_tok rows")]
    assert "c.ks[" in write and "c.vs[" in write and not [w for w in "kv" if f"__ldg(c.{w}" in write]
