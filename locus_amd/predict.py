"""Prediction from fitted models: act(X beta_vb + Z alpha_vb) for new samples, by one fit or by many at once
(a fit per cross-validation fold, cohort or tissue).  The reference returns the variational parameters and
leaves this to its user; no counterpart there.

A Predictor holds a fit's effects on the GPU in the units of the raw covariates -- the standardisation
of locus() (R/prepare_locus.R:109-141) is folded into them -- and scores samples with the fused products
(locus_amd.products): the intercept, the offset Z alpha_vb and the link function are applied in the
product's epilogue, and with many fits every sample's row meets the effects of its own fit in one call.
"""
import numpy as np

_LINKS = {"identity": "identity", "logit": "logistic", "probit": "probit"}


def _matrix(name, a, cols=None):
    a = np.asarray(a, dtype=np.float64)
    if a.ndim != 2:
        raise ValueError(f"{name} must be a matrix")
    if cols is not None and a.shape[1] != cols:
        raise ValueError(f"{name} must have {cols} columns, not {a.shape[1]}")
    return a


def _raw_effects(eff, A, rmvd):
    """Effects on standardised columns -> effects on the raw ones and the constant they leave:
    ((A - m) / s) e = A (e / s) - m' (e / s); removed columns have effect 0.  Means and deviations as scale_rm_ takes
    them, over all columns: sums over some would round otherwise.  A column of one value that is not a binary fraction
    (0.1, say) may have been kept there, its rounded mean a little off and its deviation no more than that: standardised
    it is constant, so what it adds is a constant, whatever a new sample holds."""
    keep = np.setdiff1d(np.arange(A.shape[1]), rmvd if rmvd is not None else [])
    if eff.shape[0] != len(keep):
        raise ValueError("the training covariates do not go with the fit: "
                         f"{len(keep)} columns kept, {eff.shape[0]} rows of effects")
    mean, sd = A.mean(axis=0)[keep], A.std(axis=0, ddof=1)[keep]
    if not sd.all():
        raise ValueError("the training covariates do not go with the fit: kept columns of one value: "
                         f"{keep[sd == 0].tolist()}")
    flat = (A.max(axis=0) == A.min(axis=0))[keep]
    const = ((A[0, keep] - mean) / sd)[flat] @ eff[flat]
    out = np.zeros((A.shape[1], eff.shape[1]))
    out[keep[~flat]] = eff[~flat] / sd[~flat, None]
    return out, const - mean @ out[keep]


class Predictor:
    """Predictor(vb, X, Z=None, Y=None, link="identity", ind_bin=None, single=False, device=None)

    vb: what locus() returned (not block-wise), X, Z: the training covariates as given to it.  Y: the
    training responses, for the identity link (and the continuous responses of link = "mix"), whose
    means locus() takes off; without it predictions are of the centred responses.  Lists of vb, X, Z, Y of
    equal length make a predictor of many fits of one kind.  single: effects and products in float32
    (half the memory and traffic; about 1e-6 relative to the largest terms of the linear predictor)."""

    def __init__(self, vb, X, Z=None, Y=None, link="identity", ind_bin=None, single=False, device=None):
        if link not in ("identity", "logit", "probit", "mix"):
            raise ValueError("link must be 'identity', 'logit', 'probit' or 'mix'")
        if (link == "mix") != (ind_bin is not None):
            raise ValueError("ind_bin must be given for link = 'mix' and only then")
        self.many = isinstance(vb, (list, tuple))
        lists = [[x] if not self.many else x for x in (vb, X)]
        lists += [[x] if not self.many else (x if x is not None else [None] * len(vb)) for x in (Z, Y)]
        if not lists[0] or any(len(x) != len(lists[0]) for x in lists):
            raise ValueError("vb, X, Z and Y must be lists of one length, and not empty")
        effects, consts = [], []
        for v, x, z, y in zip(*lists):
            if "beta_vb" not in v:
                raise ValueError("the fit holds no beta_vb (block-wise inference returns none)")
            beta = np.asarray(v["beta_vb"], dtype=np.float64)
            eff, const = _raw_effects(beta, _matrix("X", x), v.get("rmvd_x"))
            # locus_z_core_ has no intercept row (the responses are centred), the other links have one
            inter = 0 if link == "identity" else 1
            alpha = np.asarray(v["alpha_vb"], dtype=np.float64) if "alpha_vb" in v else np.zeros((0, beta.shape[1]))
            if alpha.shape[0] < inter:
                raise ValueError(f"the fit holds no intercept: it is not one of link = {link!r}")
            if (z is not None) != (alpha.shape[0] > inter):
                raise ValueError("Z must be given for fits with fixed covariates and only for those")
            if inter:
                const = const + alpha[0]
            if z is not None:
                za, zc = _raw_effects(alpha[inter:], _matrix("Z", z), v.get("rmvd_z"))
                eff, const = np.vstack([eff, za]), const + zc
            if y is not None:
                if link not in ("identity", "mix"):
                    raise ValueError("Y (the means that were taken off) goes with link = 'identity' or 'mix'")
                mean = _matrix("Y", y, beta.shape[1]).mean(axis=0)
                if link == "mix":
                    mean[np.asarray(ind_bin, dtype=np.int64)] = 0.0
                const = const + mean
            effects.append(eff)
            consts.append(const)
        if any(e.shape != effects[0].shape for e in effects):
            raise ValueError("the fits must have the same covariates and responses")
        z0 = lists[2][0]
        self.p = np.shape(lists[1][0])[1]
        self.q = 0 if z0 is None else np.shape(z0)[1]
        self.d = effects[0].shape[1]
        # runs of responses with one link function each, and where they go in the result
        if link == "mix":
            ind_bin = np.unique(np.asarray(ind_bin, dtype=np.int64))
            if len(ind_bin) == 0 or ind_bin[0] < 0 or ind_bin[-1] >= self.d:
                raise ValueError("ind_bin must hold indices of responses")
            parts = [("identity", np.setdiff1d(np.arange(self.d), ind_bin)), ("probit", ind_bin)]
        else:
            parts = [(_LINKS[link], np.arange(self.d))]
        import torch
        from . import device as dv
        dv.require_gpu()
        self.device = torch.device("cuda" if device is None else device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.dtype = torch.float32 if single else torch.float64
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(self.device, self.dtype)  # noqa: E731
        self.parts = [(act, torch.from_numpy(cols).to(self.device), up(np.stack([e[:, cols] for e in effects])),
                       up(np.stack([c[cols] for c in consts]))) for act, cols in parts if len(cols)]

    def score(self, A, fit=None, type="response"):
        """Device-side form: A is a GPU tensor (samples x (p + q), raw covariates, those of Z behind those
        of X) of the predictor's type; returns a GPU tensor (samples x d) and does not wait for it.
        fit: which fit scores each sample (0-based integers, on the host), for a predictor of many.  Without it the
        call can be captured into a HIP graph; with it, it cannot: the order of the samples is made on the host."""
        import torch
        from . import products
        if type not in ("response", "link"):
            raise ValueError("type must be 'response' or 'link'")
        if A.dim() != 2 or A.shape[1] != self.p + self.q:
            raise ValueError(f"A must have {self.p + self.q} columns")
        if self.many != (fit is not None):
            raise ValueError("fit must be given for a predictor of many fits and only then")
        n, groups = A.shape[0], self.parts[0][2].shape[0]
        order = off = None
        if fit is not None:
            fit = np.asarray(fit)
            if fit.size == 0:                                     # (numpy takes an empty list for floats)
                fit = fit.astype(np.int64)
            if fit.shape != (n,) or fit.dtype.kind not in "iu" or (n and not (0 <= fit.min() and fit.max() < groups)):
                raise ValueError(f"fit must hold {n} integers from 0 to {groups - 1}")
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("score() with fit cannot be captured into a graph: a replay would not see a new fit")
            order = np.argsort(fit, kind="stable")
            off = np.searchsorted(fit[order], np.arange(groups + 1))
            host = torch.empty(n + groups + 1, dtype=torch.int64, pin_memory=True)    # (a copy from other memory waits)
            host.numpy()[:] = np.concatenate([order, off])
            order, off = host.to(self.device, non_blocking=True).split([n, groups + 1])
        out = torch.empty((n, self.d), dtype=self.dtype, device=self.device)
        for act, at, B, const in self.parts:
            act = act if type == "response" else "identity"
            if fit is None:
                part = products.dense_product(A, B[0], bias=const[0], act=act)
            else:
                part = products.grouped_product(A, B, off, bias=const, act=act, gather=order)
            if fit is None and len(self.parts) == 1:
                return part
            if len(self.parts) == 1:
                out[order] = part
            else:
                out[order[:, None] if fit is not None else slice(None), at] = part
        return out

    def __call__(self, X_new, Z_new=None, fit=None, type="response"):
        """Predictions (samples x d, numpy) for raw covariates X_new (and Z_new).  type = "response": the
        mean of the responses (probabilities for binary ones); "link": the linear predictor."""
        import torch
        A = _matrix("X_new", X_new, self.p)
        if (Z_new is not None) != (self.q > 0):
            raise ValueError("Z_new must be given for fits with fixed covariates and only for those")
        if Z_new is not None:
            Z_new = _matrix("Z_new", Z_new, self.q)
            if len(Z_new) != len(A):
                raise ValueError("X_new and Z_new must have the same number of samples")
            A = np.hstack([A, Z_new])
        A = torch.from_numpy(np.ascontiguousarray(A)).to(self.device, self.dtype)
        return self.score(A, fit, type).to("cpu", torch.float64).numpy()


def predict(vb, X, X_new, Z=None, Z_new=None, Y=None, link="identity", ind_bin=None, fit=None, type="response",
            device=None):
    """One-off form: Predictor(vb, X, Z, Y, link, ind_bin)(X_new, Z_new, fit, type)."""
    return Predictor(vb, X, Z, Y, link, ind_bin, device=device)(X_new, Z_new, fit, type)
