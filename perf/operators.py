"""The operators that read a mined sample matrix, as cases to measure and compare.

A miner leaves `samples` on the GPU: one row per window, one normalised
descriptor of 32 values per template patch ([n, n_patches, 32]).  Boosting
works on that matrix:

  response   Y[r, m, h] = alpha * act(x[row r, patch m] . w[m, h] + b[m, h]) + beta * R
  rgrad      its backward pass: dW, db and the gradient of the residual R
  loss       sum of c * (softplus(z) - t z) per weak learner, with dW and db
  sample     draws of sample numbers from scores by given random numbers, after
             temperature, top-k, top-p and min-p

`run` computes them from elementary torch operations, or, with `own` set, by
the framework's kernels; `exact` computes them in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FACE_PATCHES = 608    # template patches of the 40x40 face window
PED_PATCHES = 11870   # template patches of the 64x128 pedestrian window


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _lr(op, n, p, m, h, dtype, rows=0, act="sigmoid", residual="none", name=None):
    """n samples of p patches; m weak learners with h parameter sets each;
    rows > 0: that many resampled row numbers; m < p: m patches picked."""
    c = {"op": op, "n": n, "p": p, "m": m, "h": h, "dtype": dtype, "rows": rows, "act": act,
         "residual": residual}
    return dict(c, name=name) if name else c


def _sample(b, v, s, dtype, t=1.0, k=0, p=1.0, minp=0.0, ragged=False, name=None):
    c = {"op": "sample", "b": b, "v": v, "s": s, "dtype": dtype, "t": t, "k": k, "p": p, "minp": minp,
         "ragged": ragged}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one window scored by a weak learner on every template patch: latency
        _lr("response", 1, FACE_PATCHES, FACE_PATCHES, 1, "f32", name="response-one"),
        # a stage of 37 weak learners over mined samples, added to the running score of each
        _lr("response", 4099, FACE_PATCHES, 37, 1, "f32", residual="row", name="response-stage"),
        # a boosting round: every patch's weak learner over all samples
        _lr("response", 16384, FACE_PATCHES, FACE_PATCHES, 1, "f32", residual="row", name="response-sweep"),
        # 16 regularisation strengths per patch on a resampled half-precision matrix, full residual
        _lr("response", 2000, FACE_PATCHES, FACE_PATCHES, 16, "f16", rows=2001, residual="full",
            name="response-path"),
        # backward pass of a stage's score
        _lr("rgrad", 4099, FACE_PATCHES, 37, 1, "f32", residual="row", name="rgrad-stage"),
        # backward pass over 8 parameter sets per pedestrian patch
        _lr("rgrad", 480, PED_PATCHES, PED_PATCHES, 8, "bf16", residual="full", name="rgrad-path"),
        # a fit on 960 resampled rows of a stage's samples
        _lr("loss", 960, FACE_PATCHES, FACE_PATCHES, 1, "f32", rows=960, name="loss-resampled"),
        # a fit over the whole matrix
        _lr("loss", 16384, FACE_PATCHES, FACE_PATCHES, 1, "f32", name="loss-sweep"),
        # 16 regularisation strengths per patch at once
        _lr("loss", 8191, FACE_PATCHES, FACE_PATCHES, 16, "bf16", name="loss-path"),
        # the roulette wheel over one stage's 960 samples
        _sample(1, 960, 960, "f32", name="sample-roulette"),
        # hard candidates of 32 images, a few draws from each
        _sample(32, 20011, 128, "f32", t=0.7, k=2000, p=0.95, minp=0.01, ragged=True, name="sample-pools"),
        # one large pool trimmed to its heavy part, many draws
        _sample(1, 1000003, 16384, "f32", t=0.9, k=500000, p=0.98, name="sample-large"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["response", "response", "rgrad", "loss", "loss", "sample"])
    dtype = rng.choice(["f32", "f32", "f16", "bf16"])
    if op == "sample":
        b = _log_int(rng, 1, 64)
        v = _log_int(rng, 1, 1000000 // b)
        s = _log_int(rng, 1, 16384 // b)
        return _sample(b, v, s, dtype, t=round(rng.uniform(0.3, 2.0), 3),
                       k=rng.choice([0, _log_int(rng, 1, v)]),
                       p=rng.choice([1.0, round(rng.uniform(0.05, 0.999), 4)]),
                       minp=rng.choice([0.0, round(rng.uniform(0.0001, 0.3), 5)]),
                       ragged=rng.random() < 0.5)
    p = rng.choice([FACE_PATCHES, FACE_PATCHES, PED_PATCHES])
    size = 4 if dtype == "f32" else 2
    m = p if rng.random() < 0.5 else _log_int(rng, 1, p)
    h = rng.choice([1, 1, 2, 3, 5, 8, 16, 21])
    # the matrix itself under 1.2 GB, and results under 0.15 GB
    most = min(16000, 1200000000 // (p * 32 * size), 37000000 // (m * h))
    n = _log_int(rng, 1, most)
    rows = _log_int(rng, 1, most) if rng.random() < 0.4 else 0
    residual = rng.choice(["none", "row", "full"]) if op != "loss" else "none"
    act = rng.choice(["sigmoid", "sigmoid", "none"]) if op != "loss" else "sigmoid"
    return _lr(op, n, p, m, h, dtype, rows=rows, act=act, residual=residual)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape, dtype=torch.float32):
        return torch.rand(*shape, generator=g, device="cuda", dtype=dtype)

    st = dict(case)
    if case["op"] == "sample":
        b, v = case["b"], case["v"]
        # log-weights of boosted samples; a few candidates are masked out
        scores = 2.0 * normal(b, v)
        scores.masked_fill_(uniform(b, v) < 0.03, -math.inf)
        st["scores"] = scores.to(DTYPES[case["dtype"]])
        st["u"] = uniform(b, case["s"], dtype=torch.float64)
        st["lens"] = None
        if case["ragged"]:
            st["lens"] = (v * (0.5 + 0.5 * uniform(b))).to(torch.int32).clamp_(1, v)
        return st
    n, p, m, h = case["n"], case["p"], case["m"], case["h"]
    # descriptors: non-negative cell sums, unit length, clipped, unit length again
    x = normal(n, p, 32).abs_()
    x /= x.square().sum(2, keepdim=True).sqrt_()
    x.clamp_(max=0.35355338)
    x /= x.square().sum(2, keepdim=True).sqrt_()
    st["x"] = x.to(DTYPES[case["dtype"]])
    del x
    st["w"] = 2.0 * normal(m, h, 32)
    st["b"] = 0.5 * normal(m, h)
    st["patch"] = None
    if m < p:
        st["patch"] = torch.randperm(p, generator=g, device="cuda")[:m].to(torch.int32)
    r = case["rows"] or n
    st["rows"] = None
    if case["rows"]:
        st["rows"] = torch.randint(0, n, (r,), generator=g, device="cuda", dtype=torch.int32)
    st["alpha"], st["beta"] = 0.25, 0.75  # the fourth weak learner joins a running mean
    if case["op"] == "response" and case["residual"] != "none":
        st["res"] = uniform(r) if case["residual"] == "row" else uniform(r, m, h)
    if case["op"] == "rgrad":
        st["dy"] = normal(r, m, h)
    if case["op"] == "loss":
        st["t"] = (uniform(n) < 0.4).float()
        c = torch.exp(normal(n))
        st["c"] = c / c.sum()
    return st


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------

def _picked(st):
    """The rows and patches that a call reads, as [m, r, 32] in 32 bits."""
    x = st["x"]
    if st["rows"] is not None:
        x = x[st["rows"].long()]
    if st["patch"] is not None:
        x = x[:, st["patch"].long()]
    return x.transpose(0, 1).float().contiguous()


def _logits(st, x):
    return torch.matmul(x, st["w"].transpose(1, 2).contiguous()) + st["b"][:, None, :]  # [m, r, h]


def _plain_response(st):
    y = _logits(st, _picked(st))
    if st["act"] == "sigmoid":
        y = 1.0 / (1.0 + torch.exp(-y))
    y = st["alpha"] * y.transpose(0, 1)
    if "res" in st:
        res = st["res"] if st["res"].dim() == 3 else st["res"][:, None, None]
        y = y + st["beta"] * res
    return y.contiguous()


def _plain_rgrad(st):
    x = _picked(st)
    g = st["alpha"] * st["dy"].transpose(0, 1)
    if st["act"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-_logits(st, x)))
        g = g * s * (1.0 - s)
    dw = torch.matmul(g.transpose(1, 2).contiguous(), x)
    out = {"dw": dw, "db": g.sum(1, dtype=torch.float64).float()}
    if st["residual"] == "full":
        out["dres"] = st["beta"] * st["dy"]
    elif st["residual"] == "row":
        out["dres"] = (st["beta"] * st["dy"].sum((1, 2), dtype=torch.float64)).float()
    return out


def _plain_loss(st):
    x = _picked(st)
    z = _logits(st, x)
    t, c = st["t"], st["c"]
    if st["rows"] is not None:
        t, c = t[st["rows"].long()], c[st["rows"].long()]
    t, c = t[None, :, None], c[None, :, None]
    loss = c * (torch.clamp(z, min=0) - t * z + torch.log1p(torch.exp(-z.abs())))
    g = c * (1.0 / (1.0 + torch.exp(-z)) - t)
    return {"loss": loss.sum(1, dtype=torch.float64).float(),
            "dw": torch.matmul(g.transpose(1, 2).contiguous(), x),
            "db": g.sum(1, dtype=torch.float64).float()}


def _plain_sample(st):
    s = st["scores"].double()
    b, v = s.shape
    place = torch.arange(v, device=s.device)
    usable = ~torch.isnan(s) & (s > -math.inf)
    if st["lens"] is not None:
        usable &= place < st["lens"][:, None]
    s = torch.where(usable, s, torch.full_like(s, -math.inf))
    top = s.max(1, keepdim=True).values
    w = torch.where(usable, torch.exp((s - top) / st["t"]), torch.zeros_like(s))
    s, order = torch.sort(s, dim=1, descending=True, stable=True)
    w = w.gather(1, order)
    keep = s > -math.inf
    if st["k"] > 0:
        keep &= place < st["k"]
    if st["p"] < 1.0:
        run_sum = torch.cumsum(torch.where(keep, w, torch.zeros_like(w)), 1)
        before = torch.cat([torch.zeros_like(run_sum[:, :1]), run_sum[:, :-1]], 1)
        keep &= (before < st["p"] * run_sum[:, -1:]) | (place == 0)
    keep &= w >= st["minp"]
    back = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, torch.zeros_like(w)))
    c = torch.cumsum(back, 1)
    idx = torch.searchsorted(c, st["u"] * c[:, -1:], right=True)
    last = torch.where(back > 0, place, torch.full_like(place, -1)).max(1, keepdim=True).values
    return {"index": torch.minimum(idx, last).to(torch.int32), "kept": keep.sum(1).to(torch.int32)}


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------

_trainer = None


def _own(st):
    global _trainer
    if _trainer is None:
        import surfcascade_amd
        _trainer = surfcascade_amd.Trainer(device=torch.cuda.current_device())
    tr = _trainer
    if st["op"] == "sample":
        index, kept = tr.sample(st["scores"], st["u"], temperature=st["t"], top_k=st["k"], top_p=st["p"],
                                min_p=st["minp"], lens=st["lens"])
        return {"index": index, "kept": kept}
    if st["op"] == "response":
        return tr.response(st["x"], st["w"], st["b"], patch=st["patch"], rows=st["rows"],
                           activation=st["act"], alpha=st["alpha"], residual=st.get("res"), beta=st["beta"])
    if st["op"] == "rgrad":
        dw, db, dres = tr.response_grad(st["x"], st["w"], st["dy"], st["b"], patch=st["patch"],
                                        rows=st["rows"], activation=st["act"], alpha=st["alpha"],
                                        residual=st["residual"], beta=st["beta"])
        return {"dw": dw, "db": db} if dres is None else {"dw": dw, "db": db, "dres": dres}
    loss, dw, db = tr.loss(st["x"], st["w"], st["t"], st["b"], weight=st["c"], patch=st["patch"],
                           rows=st["rows"])
    return {"loss": loss, "dw": dw, "db": db}


def run(state):
    if own:
        return _own(state)
    if state["op"] == "sample":
        return _plain_sample(state)
    if state["op"] == "response":
        return _plain_response(state)
    if state["op"] == "rgrad":
        return _plain_rgrad(state)
    return _plain_loss(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] == "sample":
        b, v, s = case["b"], case["v"], case["s"]
        size = 4 if case["dtype"] == "f32" else 2
        part = 0.75 if case["ragged"] else 1.0  # the rows' expected lengths
        return {"bytes": b * (part * v * size + s * 12 + 8), "flops": 16 * part * b * v}
    n, p, m, h = case["n"], case["p"], case["m"], case["h"]
    size = 4 if case["dtype"] == "f32" else 2
    r = case["rows"] or n
    distinct = n * (1.0 - math.exp(-r / n)) if case["rows"] else n  # rows that a resampling hits
    x = distinct * m * 32 * size + 4 * r * bool(case["rows"])
    bank = m * h * 33 * 4
    dots = 2 * 32 * r * m * h
    out = r * m * h * 4
    res = {"none": 0, "row": r * 4, "full": out}[case["residual"]]
    if case["op"] == "response":
        return {"bytes": x + bank + res + out, "flops": dots + 6 * r * m * h}
    if case["op"] == "rgrad":
        need_z = case["act"] == "sigmoid"
        return {"bytes": x + out + 2 * bank + res, "flops": (1 + need_z) * dots + 6 * r * m * h}
    return {"bytes": x + 8 * distinct + 2 * bank + m * h * 4, "flops": 2 * dots + 10 * r * m * h}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_sample(st):
    index, kept = [], []
    scores, u = st["scores"].double().cpu().numpy(), st["u"].cpu().numpy()
    lens = None if st["lens"] is None else st["lens"].cpu().numpy()
    for i, s in enumerate(scores):
        s = s[:len(s) if lens is None else lens[i]]
        pool = np.flatnonzero(s > -np.inf)  # (NaN compares false)
        ranked = pool[np.lexsort((pool, -s[pool]))]
        if len(ranked) == 0:
            index.append(np.full(u.shape[1], -1))
            kept.append(0)
            continue
        if st["k"] > 0:
            ranked = ranked[:st["k"]]
        w = np.exp((s[ranked] - s[ranked[0]]) / st["t"])
        length = len(ranked)
        if st["p"] < 1.0:
            c = np.cumsum(w)
            length = max(1, 1 + int(np.searchsorted(c, st["p"] * c[-1], side="left")))
        length = min(length, int(np.count_nonzero(w >= st["minp"])))
        chosen = ranked[:length]
        by_place = np.argsort(chosen)
        c = np.cumsum(w[:length][by_place])
        at = np.searchsorted(c, u[i] * c[-1], side="right")
        index.append(chosen[by_place][np.minimum(at, length - 1)])
        kept.append(length)
    return {"index": torch.tensor(np.array(index), dtype=torch.int32),
            "kept": torch.tensor(np.array(kept), dtype=torch.int32)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(st)
    m, h = case["m"], case["h"]
    rows = st["rows"].long() if st["rows"] is not None else torch.arange(case["n"], device="cuda")
    cols = st["patch"].long() if st["patch"] is not None else torch.arange(m, device="cuda")
    w, b = st["w"].double(), st["b"].double()
    dw, db, loss = torch.zeros_like(w), torch.zeros_like(b), torch.zeros_like(b)
    out = []
    step = max(1, 4000000 // (m * max(h, 32)))
    for i in range(0, len(rows), step):
        q = rows[i:i + step]
        x = st["x"][q[:, None], cols[None, :]].double()                       # [q, m, 32]
        z = torch.stack([(x * w[None, :, k]).sum(2) for k in range(h)], 2) + b  # [q, m, h]
        s = torch.sigmoid(z)
        if case["op"] == "response":
            y = st["alpha"] * (s if case["act"] == "sigmoid" else z)
            if case["residual"] == "row":
                y = y + st["beta"] * st["res"][i:i + step].double()[:, None, None]
            elif case["residual"] == "full":
                y = y + st["beta"] * st["res"][i:i + step].double()
            out.append(y)
            continue
        if case["op"] == "rgrad":
            g = st["alpha"] * st["dy"][i:i + step].double()
            if case["act"] == "sigmoid":
                g = g * s * torch.sigmoid(-z)
        else:
            t, c = st["t"][q].double()[:, None, None], st["c"][q].double()[:, None, None]
            # softplus(z) - t z, from the side where nothing cancels
            loss += (c * (t * torch.nn.functional.softplus(-z) + (1 - t) * torch.nn.functional.softplus(z))).sum(0)
            g = c * (s - t)
        db += g.sum(0)
        for k in range(h):
            dw[:, k] += (g[:, :, k, None] * x).sum(0)
    if case["op"] == "response":
        return torch.cat(out)
    if case["op"] == "loss":
        return {"loss": loss, "dw": dw, "db": db}
    found = {"dw": dw, "db": db}
    if case["residual"] == "full":
        found["dres"] = st["beta"] * st["dy"].double()
    elif case["residual"] == "row":
        found["dres"] = st["beta"] * st["dy"].double().sum((1, 2))
    return found
