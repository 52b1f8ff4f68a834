"""The fused and the grouped matrix products with their gradients: the cases they are timed on, their plain forms in
elementary torch operations, and the framework's calls.

A fitted model answers act(X beta + Z alpha): X holds n samples of p covariates, beta p effects on each of d responses.
  dense         C = act(alpha A B + bias) + beta residual
  dense_grad    from dC: dA, dB and the bias's gradient
  grouped       the same where consecutive runs of rows go to effects of their own (a fit per fold, cohort or tissue)
  grouped_grad  from dC: dA, dB and the bias's gradient, per run
"""
import math

import torch

own = False

F = {"f64": torch.float64, "f32": torch.float32}
ACTS = ("identity", "logistic", "probit", "softplus", "gelu", "silu")


def _dense(name, dtype, m, k, n, act, bias="column", residual=False, pre=False, colmajor=False):
    return dict(name=name, op="dense", dtype=dtype, m=m, k=k, n=n, act=act, bias=bias, residual=residual, pre=pre,
                colmajor=colmajor)


def _grouped(name, dtype, m, k, n, groups, act, residual=False, gather=False):
    return dict(name=name, op="grouped", dtype=dtype, m=m, k=k, n=n, groups=groups, act=act, residual=residual,
                gather=gather)


def listed():
    return [
        # one new individual against a small study's effects (200 samples, 500 covariates, 20 responses): latency
        _dense("one sample, small study", "f64", 1, 500, 20, "probit"),
        # one new individual against 20 000 covariates x 1000 responses: every effect is read once
        _dense("one sample", "f64", 1, 20000, 1000, "logistic"),
        # a clinic's batch of individuals, effects kept in single precision
        _dense("33 samples, single", "f32", 33, 20011, 1000, "probit"),
        # score of a logistic model at the size of the logistic workload: fitted probability minus response
        _dense("logistic score", "f64", 2000, 20000, 500, "logistic", residual=True, colmajor=True),
        # residual of 10 000 responses on the few selected covariates: the responses are read and written once
        _dense("selected covariates", "f64", 1000, 63, 10000, "identity", residual=True, colmajor=True),
        # a hidden layer over the covariates with what its backward pass needs kept
        _dense("layer kept for training", "f32", 1000, 500, 2001, "gelu", pre=True),
        # the gradients of a small study's probit model
        dict(name="probit gradient, small study", op="dense_grad", dtype="f64", m=200, k=500, n=20, act="probit"),
        # the gradients of a layer over 5000 covariates in single precision
        dict(name="layer gradient", op="dense_grad", dtype="f32", m=1999, k=5000, n=1000, act="silu"),
        # ten cross-validation folds: each sample's probability by the fit that has not seen it
        _grouped("ten folds", "f64", 1000, 5000, 501, 10, "logistic"),
        # a served batch over 64 tissues, about one individual each, some with none
        _grouped("served batch, 64 fits", "f32", 70, 2000, 200, 64, "softplus"),
        # the gradients of ten folds' fits
        dict(name="ten folds' gradient", op="grouped_grad", dtype="f64", m=1000, k=2000, n=500, groups=10,
             act="logistic", gather=False),
        # many small cohorts whose samples lie scattered in the genotype matrix
        dict(name="scattered cohorts' gradient", op="grouped_grad", dtype="f32", m=4001, k=777, n=333, groups=40,
             act="gelu", gather=True),
    ]


def draw(rng):
    def size(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    while True:
        op = rng.choice(("dense", "dense_grad", "grouped", "grouped_grad"))
        c = dict(op=op, dtype=rng.choice(("f64", "f32")), m=size(1, 4000), k=size(20, 20000), n=size(1, 10000),
                 act=rng.choice(ACTS))
        if op == "dense":
            c.update(bias=rng.choice(("none", "column", "row", "matrix")), residual=rng.random() < 0.5,
                     pre=rng.random() < 0.3, colmajor=rng.random() < 0.5)
        if op in ("grouped", "grouped_grad"):
            c.update(groups=size(2, 100), gather=rng.random() < 0.5)
        if op == "grouped":
            c.update(residual=rng.random() < 0.5)
        w = work(c)
        if w["flops"] <= 2e10 and w["bytes"] <= 1.5e8:
            return c


def work(case):
    s = 8 if case["dtype"] == "f64" else 4
    m, k, n = case["m"], case["k"], case["n"]
    used = min(case.get("groups", 1), m)
    held = case.get("groups", 1)
    if case["op"] in ("dense", "grouped"):
        outs = 1 + bool(case.get("residual")) + bool(case.get("pre")) + (case.get("bias") == "matrix")
        return {"bytes": s * (m * k + used * k * n + m * n * outs + held * n), "flops": 2.0 * m * k * n}
    return {"bytes": s * (2 * m * n + 2 * m * k + (used + held) * k * n + held * n), "flops": 4.0 * m * k * n}


def prepare(case, seed):
    dev, t = torch.device("cuda"), F[case["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    m, k, n = case["m"], case["k"], case["n"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=t)

    st = dict(case)
    rows = m
    if case.get("gather"):
        rows = m + m // 3 + 1                       # the cohorts take some of the rows, in an order of their own
        st["gather"] = torch.randperm(rows, generator=g, device=dev)[:m].contiguous()
    A = normal(k, rows).t() if case.get("colmajor") else normal(rows, k)
    st["A"] = A
    if "groups" in case:
        # group sizes as a random router gives them, uneven; the last group may be empty, others as chance has it
        G = case["groups"]
        lean = torch.rand(G, generator=g, device=dev) + 0.5
        to = torch.multinomial(lean, m, replacement=True, generator=g)
        st["offsets"] = torch.cat([to.new_zeros(1), torch.bincount(to, minlength=G).cumsum(0)])
        st["most"] = int(torch.bincount(to, minlength=G).max())
        B, b = normal(G, k, n), normal(G, n)
    else:
        B = normal(k, n)
        kind = case.get("bias", "column")
        b = {"none": lambda: None, "column": lambda: normal(n), "row": lambda: normal(m, 1),
             "matrix": lambda: normal(m, n)}[kind]()
    st["B"], st["bias"] = B / math.sqrt(k), b
    if case["op"] in ("dense", "grouped"):
        st["residual"] = torch.bernoulli(torch.full((m, n), 0.4, device=dev, dtype=t), generator=g) \
            if case.get("residual") else None
    else:
        st["dC"], st["pre"] = normal(m, n), normal(m, n)
    return st


# ---- plain forms -----------------------------------------------------------------------------------------------------

def _cdf(z):
    return 0.5 * torch.erfc(z * -math.sqrt(0.5))


def _act(name, z):
    if name == "logistic":
        return 1 / (1 + torch.exp(-z))
    if name == "probit":
        return _cdf(z)
    if name == "softplus":
        return torch.clamp(z, min=0) + torch.log1p(torch.exp(-torch.abs(z)))
    if name == "gelu":
        return z * _cdf(z)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(name, z):
    if name == "identity":
        return torch.ones_like(z)
    if name in ("probit", "gelu"):
        dens = torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
        return dens if name == "probit" else _cdf(z) + z * dens
    s = 1 / (1 + torch.exp(-z))
    if name == "softplus":
        return s
    return s * (1 - s) if name == "logistic" else s * (1 + z * (1 - s))


def _padded(st):
    """Rows of each run side by side: (groups x most) indexes of rows, which of them are rows of the run, and for every
    row its run and its place in it."""
    off, most = st["offsets"], st["most"]
    at = off[:-1, None] + torch.arange(most, device=off.device)
    valid = at < off[1:, None]
    r = torch.arange(st["m"], device=off.device)
    run_of = torch.searchsorted(off, r, right=True) - 1
    return at.clamp(max=st["m"] - 1), valid, run_of, r - off[run_of]


def _plain(st):
    A, B, act = st["A"], st["B"], st["act"]
    if st["op"] == "dense":
        z = A @ B
        if st["bias"] is not None:
            z = z + st["bias"]
        c = _act(act, z)
        if st["residual"] is not None:
            c = c - st["residual"]
        return {"C": c, "pre": z} if st["pre"] else {"C": c}
    if st["op"] == "dense_grad":
        g = st["dC"] * _slope(act, st["pre"])
        return {"dA": g @ B.t(), "dB": A.t() @ g, "dbias": g.sum(0)}
    if torch.is_tensor(st["gather"]):
        A = A[st["gather"]]
    at, valid, run_of, place = _padded(st)
    if st["op"] == "grouped":
        z = torch.bmm(A[at], B)[run_of, place] + st["bias"][run_of]
        c = _act(act, z)
        return {"C": c if st["residual"] is None else c - st["residual"]}
    g = (st["dC"] * _slope(act, st["pre"]))[at] * valid[:, :, None]
    dA = torch.bmm(g, B.transpose(1, 2).contiguous())[run_of, place]
    dB = torch.bmm(A[at].transpose(1, 2).contiguous(), g)
    return {"dA": dA, "dB": dB, "dbias": g.sum(1)}


# ---- the framework's operators ---------------------------------------------------------------------------------------

def _own(st):
    from locus_amd import products
    if st["op"] == "dense":
        if st["pre"]:
            pre = torch.empty((st["m"], st["n"]), dtype=st["A"].dtype, device=st["A"].device)
            c = products.dense_product(st["A"], st["B"], bias=st["bias"], act=st["act"], residual=st["residual"],
                                       beta=-1.0, pre=pre)
            return {"C": c, "pre": pre}
        return {"C": products.dense_product(st["A"], st["B"], bias=st["bias"], act=st["act"],
                                            residual=st["residual"], beta=-1.0)}
    if st["op"] == "dense_grad":
        dA, dB, db = products.dense_product_grad(st["dC"], st["A"], st["B"], act=st["act"], pre=st["pre"],
                                                 bias_grad="column")
        return {"dA": dA, "dB": dB, "dbias": db}
    gather = st["gather"] if torch.is_tensor(st["gather"]) else None
    if st["op"] == "grouped":
        return {"C": products.grouped_product(st["A"], st["B"], st["offsets"], bias=st["bias"], act=st["act"],
                                              residual=st["residual"], beta=-1.0, gather=gather)}
    dA, dB, db = products.grouped_product_grad(st["dC"], st["A"], st["B"], st["offsets"], act=st["act"],
                                               pre=st["pre"], gather=gather, need_bias=True)
    return {"dA": dA, "dB": dB, "dbias": db}


def run(state):
    return _own(state) if own else _plain(state)


# ---- from the definition, in 64 bits ---------------------------------------------------------------------------------

_DEFINED = {"identity": lambda z: z, "logistic": torch.sigmoid, "probit": torch.special.ndtr,
            "softplus": lambda z: torch.logaddexp(z, torch.zeros_like(z)),
            "gelu": lambda z: z * torch.special.ndtr(z), "silu": lambda z: z * torch.sigmoid(z)}


def exact(case, seed):
    st = {key: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for key, v in prepare(case, seed).items()}
    A, B, act = st["A"], st["B"], _DEFINED[st["act"]]
    if case["op"] in ("grouped", "grouped_grad"):
        edges = st["offsets"].tolist()
        runs = [(lo, hi) for lo, hi in zip(edges, edges[1:])]
        if torch.is_tensor(st["gather"]):
            A = A.index_select(0, st["gather"])
    else:
        runs, B = [(0, case["m"])], B[None]
    if case["op"] in ("dense", "grouped"):
        bias = st["bias"]
        z = torch.cat([A[lo:hi].matmul(B[i]) + (bias[i] if len(runs) > 1 else 0) for i, (lo, hi) in enumerate(runs)])
        if len(runs) == 1 and bias is not None:
            z = z + bias
        c = act(z)
        if st["residual"] is not None:
            c = c - st["residual"]
        return {"C": c, "pre": z} if case.get("pre") else {"C": c}
    pre = st["pre"].clone().requires_grad_(True)
    (g,) = torch.autograd.grad(act(pre), pre, st["dC"])
    dA = torch.cat([g[lo:hi].matmul(B[i].t().contiguous()) for i, (lo, hi) in enumerate(runs)])
    dB = torch.stack([A[lo:hi].t().contiguous().matmul(g[lo:hi]) for lo, hi in runs])
    db = torch.stack([g[lo:hi].sum(0) for lo, hi in runs])
    return {"dA": dA, "dB": dB[0], "dbias": db[0]} if case["op"] == "dense_grad" else {"dA": dA, "dB": dB, "dbias": db}
