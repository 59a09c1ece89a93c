"""The operators of an encoder layer with learned or sloped relative positions, forward and backward,
as cases that can be timed and checked: attention whose scores may be capped by a tanh, get a bias
that depends on the distance (a learned table over buckets, or a slope a head) and are masked by
document, prefix or window, with its gradients; layer norm, with its gradients.

With `own` false each operator is computed from elementary torch operations in 32 bits; with `own`
true by the library's calls (attention_bias, attention_bias_backward, layer_norm,
layer_norm_backward). Widths and lengths are this repository's: heads of 64, d = 768 and 384, a
request of 293 tokens, one sequence of 2029 to 8192 tokens, 64 requests in 18752 rows.

A case's `kind` is "attention" or "norm", `direction` "forward" or "backward". Attention: `rows`
queries over `keys` keys in `docs` documents (all of them documents of their own lengths; with fewer
queries than keys one document, the queries its last rows), `heads` and `kv_heads`, `bias` "none",
"table" (32 buckets, distances from 128 on share one a side) or "slopes", `cap` (0: none), `window`
(0: none), `mask` "document", or "prefix": the first rows of a document see each other, the others
what is before them. Norm: `rows` of `width`, `shift` whether there is a beta.
"""

import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "julia-cuda_amd")
own = False

BUCKETS, REACH = 32, 128
EPS = 1e-5
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
MOST_PAIRS = 12 * 8192 * 8192  # (query, key) pairs over all heads of the largest forward case
MOST_PAIRS_BACK = 12 * 18752 * 320


# ------------------------------------------------------------------------------ the cases
def listed():
    def att(name, direction, type, rows, keys=0, docs=1, heads=12, kv_heads=12, bias="table", cap=0.0,
            window=0, mask="document"):
        return {"name": name, "kind": "attention", "direction": direction, "type": type, "rows": rows,
                "keys": keys or rows, "docs": docs, "heads": heads, "kv_heads": kv_heads, "bias": bias,
                "cap": cap, "window": window, "mask": mask}

    def norm(name, direction, type, rows, width, shift):
        return {"name": name, "kind": "norm", "direction": direction, "type": type, "rows": rows,
                "width": width, "shift": shift}

    return [
        # one request of the mean length
        att("request", "forward", "f16", 293),
        # 64 requests concatenated into one pass
        att("batch", "forward", "f16", 18752, docs=64),
        # the longest input: a slope a head in place of a learned table
        att("long, slopes", "forward", "f16", 8192, bias="slopes"),
        # capped scores under a prefix mask, three query heads to a key head
        att("prefix, capped", "forward", "bf16", 4096, kv_heads=4, bias="none", cap=50.0, mask="prefix"),
        # the next token of a long input
        att("one row", "forward", "bf16", 1, keys=8192, kv_heads=4, bias="slopes"),
        # training on one request, on a batch of them, and on a long one
        att("request, gradients", "backward", "f16", 293),
        att("batch, gradients", "backward", "f16", 18752, docs=64),
        att("prefix, capped, gradients", "backward", "bf16", 2029, kv_heads=4, cap=50.0, mask="prefix"),
        # a layer's norm over one request and over a batch
        norm("norm of a request", "forward", "f16", 293, 768, False),
        norm("norm of a batch", "forward", "bf16", 18752, 768, True),
        norm("norm of a request, gradients", "backward", "f32", 293, 384, True),
        norm("norm of a batch, gradients", "backward", "f16", 18752, 768, True),
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.35:
        rows = log_int(rng, 1, 18752)
        return {"kind": "norm", "direction": rng.choice(["forward", "backward"]),
                "type": rng.choice(["f16", "bf16", "f32"]), "rows": rows,
                "width": rng.choice([64, 384, 768, 1152, 1536, log_int(rng, 8, 2048), 8 * log_int(rng, 2, 256)]),
                "shift": rng.random() < 0.5}
    while True:
        direction = rng.choice(["forward", "backward"])
        kv_heads = rng.choice([1, 2, 4, 6, 12])
        heads = kv_heads * rng.choice([1, 1, 2, 3])
        docs = rng.choice([1, 1, 1, log_int(rng, 2, 64)])
        rows = log_int(rng, 1, 8192 if docs == 1 else 18752)
        keys = rows
        if direction == "forward" and docs == 1 and rng.random() < 0.3:
            rows, keys = log_int(rng, 1, 64), log_int(rng, 64, 16384)
        if rows < docs or heads > 16:
            continue
        case = {"kind": "attention", "direction": direction, "type": rng.choice(["f16", "bf16"]),
                "rows": rows, "keys": keys, "docs": docs, "heads": heads, "kv_heads": kv_heads,
                "bias": rng.choice(["none", "table", "table", "slopes"]),
                "cap": rng.choice([0.0, 0.0, 30.0, 50.0]), "window": rng.choice([0, 0, 0, 64]),
                "mask": rng.choice(["document", "document", "prefix"])}
        longest = max(lengths(case))
        pairs = heads * longest * (longest if rows == keys else rows) * docs
        if pairs <= (MOST_PAIRS if direction == "forward" else MOST_PAIRS_BACK):
            return case


def lengths(case):
    """The documents' lengths: the same for every pass of a case, by its sizes alone. They spread
    about 2:1 around the mean."""
    docs, keys = case["docs"], case["keys"]
    r = random.Random(1000003 * docs + keys)
    share = [r.uniform(0.6, 1.4) for _ in range(docs)]
    total, out, at = sum(share), [], 0.0
    ends = []
    for s in share:
        at += s
        ends.append(int(round(at / total * keys)))
    ends[-1] = keys
    prev = 0
    for i, e in enumerate(ends):
        e = max(prev + 1, min(e, keys - (docs - 1 - i)))  # every document has a row
        out.append(e - prev)
        prev = e
    return out


def spans(case):
    """Each query's keys [first, one past last), as global key rows, without the window."""
    out, at = [], 0
    for n in lengths(case):
        prefix = (n + 2) // 3
        for i in range(n):
            out.append((at, at + n if case["mask"] == "document" else at + max(i + 1, prefix)))
        at += n
    return out[len(out) - case["rows"]:]


def pairs(case):
    """Unmasked (query, key) pairs of a head."""
    first, w, total = case["keys"] - case["rows"], case["window"], 0
    for i, (lo, hi) in enumerate(spans(case)):
        if w:
            lo, hi = max(lo, first + i - w), min(hi, first + i + w + 1)
        total += max(0, hi - lo)
    return total


def work(case):
    if case["kind"] == "norm":
        size, n, d = (4 if case["type"] == "f32" else 2), case["rows"], case["width"]
        if case["direction"] == "forward":
            return {"bytes": 2 * size * n * d + 4 * d * (2 if case["shift"] else 1) + 8 * n, "flops": 8 * n * d}
        return {"bytes": 3 * size * n * d + 4 * d * (3 if case["shift"] else 2) + 8 * n, "flops": 12 * n * d}
    d, dk, nq, nk, h = 64 * case["heads"], 64 * case["kv_heads"], case["rows"], case["keys"], case["heads"]
    table = 4 * BUCKETS * h if case["bias"] == "table" else 0
    if case["direction"] == "forward":
        return {"bytes": 2 * (2 * nq * d + 2 * nk * dk) + 4 * nq * h + table + 8 * nq, "flops": 4 * 64 * h * pairs(case)}
    # read q, k, v, the outputs, their gradient and the log-sums; written dq, dk, dv
    return {"bytes": 2 * (4 * nq * d + 4 * nk * dk) + 4 * nq * h + 2 * table + 8 * nq,
            "flops": 10 * 64 * h * pairs(case)}


# ------------------------------------------------------------------------------ what a program has in hand
def buckets(reach=REACH, count=BUCKETS):
    """The bucket of each distance key - query from -reach to reach: half of them for keys after the
    query; in each half the first half for one distance each, the others over logarithmic ranges
    that end at `reach`."""
    half, exact = count // 2, count // 4
    out = []
    for dist in range(-reach, reach + 1):
        a = abs(dist)
        if a >= exact:
            # floor of log(a / exact) / log(reach / exact) (half - exact), in whole numbers
            step = 0
            while step + 1 < half - exact and a ** (half - exact) * exact ** (step + 1) >= \
                    reach ** (step + 1) * exact ** (half - exact):
                step += 1
            a = exact + step
        out.append(a + (half if dist > 0 else 0))
    return out


def gaussian(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["type"]]
    s = {"case": case}
    if case["kind"] == "norm":
        n, d = case["rows"], case["width"]
        # a residual stream: a mean off zero and a few wide columns
        width = 1.0 + 3.0 * (gaussian(gen, d) > 2.0)
        s["x"] = (gaussian(gen, n, d) * width + 0.3 * gaussian(gen, d)).to(t)
        s["gamma"] = 1.0 + 0.2 * gaussian(gen, d)
        s["beta"] = 0.1 * gaussian(gen, d) if case["shift"] else None
        s["stats"] = torch.empty(n, 2, device="cuda")
        if case["direction"] == "backward":
            s["dy"] = (0.05 * gaussian(gen, n, d)).to(t)
            x = s["x"].double()
            mean = x.mean(1)
            var = (x - mean[:, None]).square().mean(1)
            s["stats"] = torch.stack((mean, 1.0 / torch.sqrt(var + EPS)), 1).float().contiguous()
            s["dx"], s["dgamma"] = torch.empty_like(s["x"]), torch.empty(d, device="cuda")
            s["dbeta"] = torch.empty(d, device="cuda") if case["shift"] else None
        else:
            s["y"] = torch.empty_like(s["x"])
        return own_norm(s) if own else s

    nq, nk, h, g = case["rows"], case["keys"], case["heads"], case["kv_heads"]
    qkv = gaussian(gen, nk, (h + 2 * g) * 64)
    qkv[:, : (h + g) * 64] *= 1.3  # scores of a deviation of about 1.7
    s["qkv"] = qkv.to(t)
    s["q"] = s["qkv"][nk - nq:, : h * 64]
    s["k"], s["v"] = s["qkv"][:, h * 64:(h + g) * 64], s["qkv"][:, (h + g) * 64:]
    s["span"] = torch.tensor(spans(case), dtype=torch.int32, device="cuda")
    s["table"] = s["bucket"] = s["slopes"] = None
    if case["bias"] == "table":
        s["table"] = gaussian(gen, BUCKETS, h)
        s["bucket"] = torch.tensor(buckets(), dtype=torch.int32, device="cuda")
    elif case["bias"] == "slopes":
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda") / h)
    # the documents' rows side by side, for the plain form: row i of document b, or row 0 again
    lens = lengths(case)
    most = max(lens)
    at = torch.tensor([0] + lens, device="cuda").cumsum(0)
    i = torch.arange(most, device="cuda")
    length = torch.tensor(lens, device="cuda")
    s["key_real"] = i[None] < length[:, None]
    s["key_rows"] = torch.where(s["key_real"], at[:-1, None] + i[None], 0)
    first = nk - nq
    if first:
        s["query_rows"] = torch.arange(nq, device="cuda")[None]
        s["query_real"] = torch.ones(1, nq, dtype=torch.bool, device="cuda")
    else:
        s["query_rows"], s["query_real"] = s["key_rows"], s["key_real"]
    s["query_back"] = s["query_real"].flatten().nonzero()[:, 0]
    s["key_back"] = s["key_real"].flatten().nonzero()[:, 0]
    s["o"] = torch.empty(nq, h * 64, dtype=t, device="cuda")
    s["lse"] = torch.empty(h, nq, device="cuda")
    if case["direction"] == "backward":
        o, s["lse"] = plain_forward(s)
        s["o"] = o.to(t)
        s["dout"] = (0.02 * gaussian(gen, nq, h * 64)).to(t)
        s["dqkv"] = torch.empty_like(s["qkv"])
        s["dtable"] = torch.empty_like(s["table"]) if s["table"] is not None else None
    return own_attention(s) if own else s


def run(s):
    back = s["case"]["direction"] == "backward"
    if s["case"]["kind"] == "norm":
        if own:
            return call_norm_backward(s) if back else call_norm(s)
        return plain_norm_backward(s) if back else plain_norm(s)
    if own:
        return call_attention_backward(s) if back else call_attention(s)
    if back:
        return plain_backward(s)
    o, lse = plain_forward(s)
    return {"o": o.to(s["q"].dtype), "lse": lse}


# ------------------------------------------------------------------------------ the library's calls
def library():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    import julia_hip

    return julia_hip


def pointer(t):
    return 0 if t is None else t.data_ptr()


def own_norm(s):
    jh = library()
    s["jh"], s["dtype"] = jh, s["case"]["type"]
    s["stream"] = torch.cuda.current_stream().cuda_stream
    n, d = s["x"].shape
    if s["case"]["direction"] == "backward":
        s["scratch"] = jh.Scratch(*jh.layer_norm_scratch(n, d))
    return s


def own_attention(s):
    """The arguments' block and the scratch that a program makes once for its buffers."""
    jh = library()
    c = s["case"]
    stride = s["qkv"].stride(0)
    s["jh"] = jh
    s["stream"] = torch.cuda.current_stream().cuda_stream
    s["args"] = jh.attention_bias_args(
        c["type"], pointer(s["q"]), pointer(s["k"]), pointer(s["v"]), pointer(s["o"]), c["rows"], c["keys"],
        c["heads"], c["kv_heads"], q_stride=stride, kv_stride=stride, q_first=c["keys"] - c["rows"],
        scale=0.125, cap=c["cap"], table=pointer(s["table"]), bucket=pointer(s["bucket"]), buckets=BUCKETS,
        reach=REACH, slopes=pointer(s["slopes"]), window=c["window"], span=pointer(s["span"]),
        lse=pointer(s["lse"]))
    back = c["direction"] == "backward"
    s["scratch"] = jh.Scratch(*jh.attention_bias_scratch(s["args"], backward=back))
    if back:
        e = s["dqkv"].element_size()
        dq = s["dqkv"].data_ptr()
        dk = dq + 64 * c["heads"] * e
        s["grads"] = jh.attention_bias_grads(
            s["args"], s["dout"].data_ptr(), dq, dk, dk + 64 * c["kv_heads"] * e, dq_stride=stride, dkv_stride=stride,
            dtable=pointer(s["dtable"]))
    return s


def call_attention(s):
    s["jh"].attention_bias(s["args"], scratch=s["scratch"], stream=s["stream"])
    return {"o": s["o"], "lse": s["lse"]}


def call_attention_backward(s):
    s["jh"].attention_bias_backward(s["args"], s["grads"], scratch=s["scratch"], stream=s["stream"])
    return {"dqkv": s["dqkv"]} if s["dtable"] is None else {"dqkv": s["dqkv"], "dtable": s["dtable"]}


def call_norm(s):
    n, d = s["x"].shape
    s["jh"].layer_norm(s["dtype"], s["x"].data_ptr(), n, d, s["gamma"].data_ptr(), pointer(s["beta"]), EPS,
                       s["y"].data_ptr(), stats=s["stats"].data_ptr(), stream=s["stream"])
    return {"y": s["y"], "stats": s["stats"]}


def call_norm_backward(s):
    n, d = s["x"].shape
    s["jh"].layer_norm_backward(s["dtype"], s["x"].data_ptr(), s["dy"].data_ptr(), n, d, s["gamma"].data_ptr(),
                                s["stats"].data_ptr(), s["dx"].data_ptr(), s["dgamma"].data_ptr(),
                                pointer(s["dbeta"]), scratch=s["scratch"], stream=s["stream"])
    out = {"dx": s["dx"], "dgamma": s["dgamma"]}
    return out if s["dbeta"] is None else {**out, "dbeta": s["dbeta"]}


# ------------------------------------------------------------------------------ the plain forms
def plain_norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    off = x - mean
    rstd = 1.0 / torch.sqrt((off * off).mean(1, keepdim=True) + EPS)
    y = off * rstd * s["gamma"]
    if s["beta"] is not None:
        y = y + s["beta"]
    return {"y": y.to(s["x"].dtype), "stats": torch.cat((mean, rstd), 1)}


def plain_norm_backward(s):
    dy, mean, rstd = s["dy"].float(), s["stats"][:, :1], s["stats"][:, 1:]
    xh = (s["x"].float() - mean) * rstd
    g = dy * s["gamma"]
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    out = {"dx": dx.to(s["x"].dtype), "dgamma": (dy * xh).sum(0)}
    return out if s["dbeta"] is None else {**out, "dbeta": dy.sum(0)}


def by_head(x, rows, heads, repeat):
    """The [documents][heads][rows][64] of [rows][heads 64], each head `repeat` times."""
    x = x.float()[rows].unflatten(2, (heads, 64)).transpose(1, 2)
    return x.repeat_interleave(repeat, 1) if repeat > 1 else x


def distances(s):
    c = s["case"]
    i = torch.arange(s["query_rows"].shape[1], device="cuda") + (c["keys"] - c["rows"])
    return torch.arange(s["key_rows"].shape[1], device="cuda")[None] - i[:, None]


def unmasked(s, dist):
    lo, hi = s["span"][s["query_rows"]].long().unbind(2)
    j = s["key_rows"][:, None]
    ok = (j >= lo[..., None]) & (j < hi[..., None]) & s["key_real"][:, None] & s["query_real"][..., None]
    if s["case"]["window"]:
        ok = ok & (dist.abs() <= s["case"]["window"])
    return ok[:, None]


def plain_scores(s):
    """(scores with masked ones -inf, the tanh of the cap or None, the mask)"""
    c = s["case"]
    each = c["heads"] // c["kv_heads"]
    q = by_head(s["q"], s["query_rows"], c["heads"], 1)
    k = by_head(s["k"], s["key_rows"], c["kv_heads"], each)
    sc, tanh = torch.matmul(q, k.transpose(2, 3).contiguous()) * 0.125, None
    if c["cap"]:
        tanh = torch.tanh(sc / c["cap"])
        sc = tanh * c["cap"]
    dist = distances(s)
    if c["bias"] == "table":
        sc = sc + s["table"][s["bucket"].long()[dist.clamp(-REACH, REACH) + REACH]].permute(2, 0, 1)
    elif c["bias"] == "slopes":
        sc = sc - s["slopes"][:, None, None] * dist.abs()
    ok = unmasked(s, dist)
    return sc.masked_fill(~ok, -math.inf), tanh, ok


def rows_back(x, back):
    """[documents][heads][rows][64] as [rows][heads 64], the documents end to end."""
    return x.transpose(1, 2).flatten(2).flatten(0, 1)[back]


def plain_forward(s):
    c = s["case"]
    sc = plain_scores(s)[0]
    top = sc.amax(3, keepdim=True).clamp_min(-3e38)
    p = torch.exp(sc - top)
    del sc
    total = p.sum(3, keepdim=True)
    v = by_head(s["v"], s["key_rows"], c["kv_heads"], c["heads"] // c["kv_heads"])
    o = torch.matmul(p, v) / total.clamp_min(1e-38)
    lse = torch.where(total > 0, top + torch.log(total), -math.inf)[..., 0]
    return rows_back(o, s["query_back"]), lse.transpose(0, 1).flatten(1)[:, s["query_back"]].contiguous()


def plain_backward(s):
    c = s["case"]
    each = c["heads"] // c["kv_heads"]
    sc, tanh, ok = plain_scores(s)
    lse = s["lse"][:, s["query_rows"]].transpose(0, 1)
    p = torch.where(ok, torch.exp(sc - lse[..., None]), 0.0)
    del sc
    q = by_head(s["q"], s["query_rows"], c["heads"], 1)
    do = by_head(s["dout"], s["query_rows"], c["heads"], 1)
    o = by_head(s["o"], s["query_rows"], c["heads"], 1)
    v = by_head(s["v"], s["key_rows"], c["kv_heads"], each)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = p * (ds - (do * o).sum(3, keepdim=True))
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    del p
    out = {}
    if s["dtable"] is not None:
        # the sum along each diagonal: rows of one more than their length put it in a column
        h, nq, nk = ds.shape[1:]
        w = nq + nk - 1
        a = torch.nn.functional.pad(ds.sum(0).flip(1), (0, nq)).flatten(1)[:, : nq * w].unflatten(1, (nq, w))
        a = a.sum(1, dtype=torch.float64)
        first = c["keys"] - c["rows"]
        b = s["bucket"].long()[(torch.arange(w, device="cuda") - (nq - 1) - first).clamp(-REACH, REACH) + REACH]
        out["dtable"] = torch.matmul((b[None] == torch.arange(BUCKETS, device="cuda")[:, None]).double(),
                                     a.transpose(0, 1)).float()
    if tanh is not None:
        ds = ds * (1.0 - tanh * tanh)
    ds = ds * 0.125
    k = by_head(s["k"], s["key_rows"], c["kv_heads"], each)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    if each > 1:
        dk, dv = (x.unflatten(1, (c["kv_heads"], each)).sum(2) for x in (dk, dv))
    out["dqkv"] = torch.cat((rows_back(dq, s["query_back"]), rows_back(dk, s["key_back"]),
                             rows_back(dv, s["key_back"])), 1).to(s["q"].dtype)
    return out


# ------------------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return exact_norm(s)
    n, h, each = case["rows"], case["heads"], case["heads"] // case["kv_heads"]
    q, k, v = (s[x].double().reshape(len(s[x]), -1, 64) for x in "qkv")
    back = case["direction"] == "backward"
    o, lse = torch.empty_like(q), torch.empty(h, n, dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros_like(x) for x in (q, k, v))
    dt = torch.zeros(BUCKETS, h, dtype=torch.float64, device="cuda")
    at, first = 0, case["keys"] - n
    for length in lengths(case):
        rq = slice(at, at + length) if not first else slice(0, n)
        rk = slice(at, at + length)
        j = torch.arange(at, at + length, device="cuda")
        i = j if not first else torch.arange(first, first + n, device="cuda")
        away = j[None] - i[:, None]
        ok = (j[None] >= s["span"][rq, 0][:, None]) & (j[None] < s["span"][rq, 1][:, None])
        if case["window"]:
            ok &= away.abs() <= case["window"]
        if case["bias"] == "table":
            which = s["bucket"].long()[torch.clamp(away, -REACH, REACH) + REACH]
        for x in range(h):
            y = x // each
            a = (q[rq, x] @ k[rk, y].T) / 8.0
            slope = torch.ones_like(a)
            if case["cap"]:
                a = case["cap"] * torch.tanh(a / case["cap"])
                slope = 1.0 - (a / case["cap"]) ** 2
            if case["bias"] == "table":
                a = a + s["table"].double()[which, x]
            elif case["bias"] == "slopes":
                a = a - s["slopes"].double()[x] * away.abs()
            a[~ok] = -math.inf
            if not back:
                lse[x, rq] = torch.logsumexp(a, 1)
                o[rq, x] = torch.softmax(a, 1).nan_to_num(0.0) @ v[rk, y]
                continue
            p = torch.exp(a - s["lse"].double()[x, rq][:, None]).masked_fill(~ok, 0.0)
            g = s["dout"][rq, 64 * x:64 * x + 64].double()
            d = (g * s["o"][rq, 64 * x:64 * x + 64].double()).sum(1, keepdim=True)
            ds = p * (g @ v[rk, y].T - d)
            dv[rk, y] += p.T @ g
            if case["bias"] == "table":
                # along the diagonals: the columns of a skewed copy
                m = len(j)
                skew = torch.zeros(len(i), len(i) + m, dtype=torch.float64, device="cuda")
                skew[:, :m] = ds.flip(0)
                skew = skew.reshape(-1)[: len(i) * (len(i) + m - 1)].reshape(len(i), -1).sum(0)
                far = torch.arange(len(skew), device="cuda") - (len(i) - 1) + int(j[0] - i[0])
                dt[:, x].index_add_(0, s["bucket"].long()[far.clamp(-REACH, REACH) + REACH], skew)
            ds = ds * slope / 8.0
            dq[rq, x] += ds @ k[rk, y]
            dk[rk, y] += ds.T @ q[rq, x]
        at += length
    if not back:
        return {"o": o.flatten(1), "lse": lse}
    out = {"dqkv": torch.cat((dq.flatten(1), dk.flatten(1), dv.flatten(1)), 1)}
    return {**out, "dtable": dt} if case["bias"] == "table" else out


def exact_norm(s):
    x, gamma = s["x"].double(), s["gamma"].double()
    if s["case"]["direction"] == "forward":
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + EPS) * gamma
        return {"y": y if s["beta"] is None else y + s["beta"].double(),
                "stats": torch.cat((mean, (var + EPS) ** -0.5), 1)}
    dy, mean, rstd = s["dy"].double(), s["stats"][:, :1].double(), s["stats"][:, 1:].double()
    xh = (x - mean) * rstd
    t = dy * gamma
    dx = (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True)) * rstd
    out = {"dx": dx, "dgamma": (dy * xh).sum(0)}
    return out if s["dbeta"] is None else {**out, "dbeta": dy.sum(0)}
