"""CPU tests of the biased attention's and layer norm's host side: the buckets and spans a program
makes for them, the checks of their arguments, and the scratch they ask for. And of the formulas
that the GPU tests hold the kernels to: against torch's own differentiation in 64 bits."""

import math

import numpy as np
import pytest
import torch

import julia_hip as jh
import relative as R


def exact_bucket(t, buckets, most, both):
    """In whole numbers: a is in range r of a side's m when (a / e)^m >= (most / e)^r."""
    side = buckets // 2 if both else buckets
    e = side // 2
    m = side - e
    a = abs(t) if both else max(-t, 0)
    if a >= e:
        r = 0
        while r + 1 < m and a ** m * e ** (r + 1) >= most ** (r + 1) * e ** m:
            r += 1
        a = e + r
    return a + (side if both and t > 0 else 0)


@pytest.mark.parametrize("buckets,most,both,reach", [(32, 128, True, 128), (32, 128, False, 128), (64, 512, True, 512),
                                                      (8, 20, True, 40), (2, 2, False, 5), (6, 3, True, 7),
                                                      (32, 128, True, 0), (128, 256, False, 300)])
def test_relative_buckets(buckets, most, both, reach):
    got = jh.relative_buckets(buckets, most, both, reach)
    want = [exact_bucket(t, buckets, most, both) for t in range(-reach, reach + 1)]
    assert got.tolist() == want
    assert got.min() >= 0 and got.max() < buckets


def test_relative_buckets_refusals():
    for args, why in [((3, 128, True, 4), "even"), ((1, 128, False, 4), "at least 2"), ((32, 8, True, 4), "max_distance"),
                      ((32, 128, True, 513), "reach"), ((32, 128, True, -1), "reach"), ((2048, 4096, True, 4), "1024")]:
        with pytest.raises(jh.JuliaHipError, match=why):
            jh.relative_buckets(*args)


def test_spans():
    assert jh.spans([2, 0, 3]).tolist() == [[0, 2], [0, 2], [2, 5], [2, 5], [2, 5]]
    assert jh.spans([2, 3], [0, 2]).tolist() == [[0, 1], [0, 2], [2, 4], [2, 4], [2, 5]]
    assert jh.spans([]).shape == (0, 2)
    for args, why in [(([2], [3]), "longer"), (([2], [1, 1]), "prefixes"), (([1 << 30],), "2\\^30")]:
        with pytest.raises((jh.JuliaHipError, MemoryError), match=why):
            if args == ([1 << 30],):
                n = np.array([1 << 30], np.uintp)
                out = np.empty((1, 2), np.int32)
                jh._call(jh.lib().julia_hip_prep_spans, jh._np_ptr(n), None, 1, jh._np_ptr(out))
            else:
                jh.spans(*args)


def args(**kw):
    a = dict(type="f16", q=4096, k=4096, v=4096, o=4096, nq=10, nk=10, heads=4, kv_heads=2, lse=4096)
    return jh.attention_bias_args(**{**a, **kw})


def grads(a, **kw):
    g = dict(dout=4096, dq=4096, dk=4096, dv=4096)
    return jh.attention_bias_grads(a, **{**g, **kw})


REFUSED = [(dict(nq=-1), "queries"), (dict(nk=1 << 30), "keys"), (dict(heads=0, kv_heads=1), "heads"),
           (dict(heads=5), "heads"), (dict(heads=257, kv_heads=257), "heads"), (dict(q_first=-1), "q_first"),
           (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"),
           (dict(scale=math.inf), "scale"), (dict(cap=-1.0), "cap"), (dict(cap=0.01, scale=100.0), "caps"), (dict(cap=math.nan), "cap"),
           (dict(window=-1), "window"), (dict(table=4, bucket=4, buckets=2, slopes=4), "not both"),
           (dict(table=4, buckets=2), "buckets"), (dict(table=4, bucket=4, buckets=0), "buckets"),
           (dict(table=4, bucket=4, buckets=2, reach=513), "reach"), (dict(table=4, bucket=4, buckets=2, reach=-1), "reach"),
           (dict(table=4, bucket=4, buckets=2, reach=512, heads=32, kv_heads=1), "too long"),
           (dict(table=2, bucket=4, buckets=2), "aligned"), (dict(slopes=2), "aligned"), (dict(span=4), "aligned"),
           (dict(q=0), "q must"), (dict(k=4098), "k must"), (dict(v=0), "v must"), (dict(o=4104), "o must"),
           (dict(q_stride=255), "apart"), (dict(q_stride=260), "apart"), (dict(kv_stride=120), "apart"),
           (dict(o_stride=1 << 23), "apart"), (dict(lse=2), "lse"),
           (dict(nq=1 << 24, heads=256, kv_heads=256), "rows"), (dict(nk=1 << 29, heads=4, kv_heads=4), "keys of heads")]


@pytest.mark.parametrize("kw,why", REFUSED, ids=[str(k) for k, _ in REFUSED])
def test_attention_refusals(kw, why):
    with pytest.raises(jh.JuliaHipError, match=why):
        jh.attention_bias_check(args(**kw))
    # the calls themselves, which would not reach a GPU here either
    with pytest.raises(jh.JuliaHipError, match=why):
        jh.attention_bias(args(**kw))


def test_attention_gradients_refusals():
    ok = args()
    jh.attention_bias_check(ok)
    jh.attention_bias_check(ok, grads(ok))
    bad = jh.attention_bias_args("f16", 4096, 4096, 4096, 4096, 10, 10, 4)
    bad.type = 2
    with pytest.raises(jh.JuliaHipError, match="f16 or bf16"):
        jh.attention_bias_check(bad)
    for a, g, why in [(args(lse=0), {}, "lse"), (ok, dict(dout=0), "dout"),
                      (ok, dict(dq=8), "dq"), (ok, dict(dk=0), "dk"), (ok, dict(dv=0), "dv"),
                      (ok, dict(dtable=4096), "dtable"), (args(table=4, bucket=4, buckets=2), {}, "dtable"),
                      (ok, dict(dkv_stride=100), "apart"), (ok, dict(do_stride=8), "apart")]:
        with pytest.raises(jh.JuliaHipError, match=why):
            jh.attention_bias_check(a, grads(a, **g))
    # no queries, or no keys: their buffers may be null
    none = args(nq=0, q=0, o=0, lse=0)
    jh.attention_bias_check(none, grads(none, dout=0, dq=0))
    none = args(nk=0, k=0, v=0)
    jh.attention_bias_check(none, grads(none, dk=0, dv=0))


def test_scratch_sizes():
    """A grid that fills the GPU needs none; few rows over many keys need their tiles' parts."""
    assert jh.attention_bias_scratch(args(nq=20000, nk=20000)) == (0, 0)
    floats, counters = jh.attention_bias_scratch(args(nq=1, nk=8192))
    assert counters == 2 and floats > 0
    floats, counters = jh.attention_bias_scratch(args(nq=1000, nk=1000), backward=True)
    assert floats >= 2 * 4 * 1000 and counters == 0
    assert jh.layer_norm_scratch(0, 8)[0] >= 0 and jh.layer_norm_scratch(1000, 768)[0] > 0


NORM_REFUSED = [(dict(rows=-1), "rows"), (dict(d=0), "values"), (dict(d=8193), "values"), (dict(x=0), "x must"),
                (dict(x=4097), "x must"), (dict(y=0), "y must"), (dict(gamma=0), "gamma"), (dict(beta=2), "beta"),
                (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(stats=4), "stats"), (dict(x_stride=7), "apart")]


@pytest.mark.parametrize("kw,why", NORM_REFUSED, ids=[str(k) for k, _ in NORM_REFUSED])
def test_layer_norm_refusals(kw, why):
    a = dict(type="f16", x=4096, rows=4, d=8, gamma=4096, beta=4096, eps=1e-5, y=4096, stats=4096)
    with pytest.raises(jh.JuliaHipError, match=why):
        jh.layer_norm(**{**a, **kw})


def test_layer_norm_gradients_refusals():
    a = dict(type="f32", x=4096, dy=4096, rows=4, d=8, gamma=4096, stats=4096, dx=4096, dgamma=4096, dbeta=4096)
    for kw, why in [(dict(dy=0), "dy must"), (dict(dy=4098), "dy must"), (dict(dx=0), "dx must"), (dict(stats=0), "stats"),
                    (dict(dgamma=0), "dgamma"), (dict(dbeta=6), "dbeta"), (dict(dy_stride=3), "apart"), (dict(), "scratch")]:
        with pytest.raises(jh.JuliaHipError, match=why):
            jh.layer_norm_backward(**{**a, **kw})


def test_the_formulas_are_those_of_differentiation():
    """tests/relative.py's gradients against torch's own, in 64 bits."""
    g = torch.Generator().manual_seed(0)
    n, heads, kv = 40, 4, 2
    q, k, v = (torch.randn(n, h, 64, generator=g, dtype=torch.float64).requires_grad_() for h in (heads, kv, kv))
    table = torch.randn(32, heads, generator=g, dtype=torch.float64).requires_grad_()
    bucket = torch.from_numpy(jh.relative_buckets(32, 16, reach=16))
    span = torch.from_numpy(jh.spans([25, 15], [9, 3]))
    dout = torch.randn(n, heads, 64, generator=g, dtype=torch.float64)
    out = R.attention(q.detach(), k.detach(), v.detach(), cap=3.0, table=table.detach(), bucket=bucket, reach=16, span=span,
                      window=20, dout=dout)
    t = torch.arange(n)[None] - torch.arange(n)[:, None]
    a = torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(2, 1)) / 8
    a = 3.0 * torch.tanh(a / 3.0) + table[bucket.long()[t.clamp(-16, 16) + 16]].permute(2, 0, 1)
    j = torch.arange(n)
    ok = (j[None] >= span[:, :1]) & (j[None] < span[:, 1:]) & (t.abs() <= 20)
    p = torch.softmax(a.masked_fill(~ok, -math.inf), 2)
    o = torch.einsum("hij,jhd->ihd", p, v.repeat_interleave(2, 1))
    o.backward(dout)
    for x, y in (("o", o.detach()), ("dq", q.grad), ("dk", k.grad), ("dv", v.grad), ("dtable", table.grad)):
        assert float((out[x] - y).abs().max()) < 1e-12, x
    x = torch.randn(9, 30, generator=g, dtype=torch.float64).requires_grad_()
    gamma, beta = (torch.randn(30, generator=g, dtype=torch.float64).requires_grad_() for _ in range(2))
    dy = torch.randn(9, 30, generator=g, dtype=torch.float64)
    y = torch.nn.functional.layer_norm(x, (30,), gamma, beta, 1e-5)
    y.backward(dy)
    out = R.norm(x.detach(), gamma.detach(), beta.detach(), 1e-5, dy)
    for key, want in (("y", y.detach()), ("dx", x.grad), ("dgamma", gamma.grad), ("dbeta", beta.grad)):
        assert float((out[key] - want).abs().max()) < 1e-12, key
