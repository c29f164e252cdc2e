"""
The read-out of several latent fields, as it is measured: standardisation (layer norm) and the log probability of
observed classes under a linear read-out (softmax cross entropy), each with its reverse mode.

``run`` computes the operators from elementary torch operations where ``own`` is false and calls this package
(:mod:`gptools_amd.glm`) where it is true. Formulas, for one row x of length n (a token's features, or a whole lattice):

    layer_norm        mean = sum x / n,  var = sum (x - mean)^2 / n,  rstd = 1 / sqrt(var + eps),  h = (x - mean) rstd
                      y = h w + b
    layer_norm_vjp    g = ybar w,  xbar = rstd (g - <g> - h <g h>),  wbar = sum_rows ybar h,  bbar = sum_rows ybar
    categorical_logit_glm_lpmf       eta_v = alpha_v + beta_v . x,  lp = eta_y - log sum_v exp eta_v,  0 where y < 0
    categorical_logit_glm_lpmf_vjp   r_v = lpbar ([v = y] - softmax(eta)_v),  xbar = sum_v r_v beta_v,
                                     alphabar = sum_rows r,  betabar_v = sum_rows r_v x
"""
import torch

own = False

TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5


def _norm(name, op, dtype, rows, height, width, affine=True):
    # height == 1: rows of `width` features, else lattices of height x width that are standardised as a whole
    return {"name": name, "op": op, "type": dtype, "rows": rows, "height": height, "width": width, "affine": affine}


def _class(name, op, dtype, rows, features, classes, masked=0.0, mean=False):
    # masked: the share of rows without an observation; mean: the cotangent of a mean over the observed rows' losses
    # (a training step), else that of a sum of log probabilities (a sampler's log density)
    return {"name": name, "op": op, "type": dtype, "rows": rows, "features": features, "classes": classes,
            "masked": masked, "mean": mean}


def listed():
    return [
        # one token of a generating model: the smallest call, latency alone
        _norm("norm_one_token", "norm", "bf16", 1, 1, 4096),
        # the tokens of a training batch, forward and backward: many rows of ordinary length
        _norm("norm_tokens", "norm", "bf16", 16384, 1, 4096),
        _norm("norm_grad_tokens", "norm_grad", "bf16", 16384, 1, 4096),
        # an odd number of rows of an odd length: no row but the first is aligned
        _norm("norm_grad_odd", "norm_grad", "f32", 8191, 1, 1001),
        # bench.py's launch of 16 lattices of 4096 x 4096, each standardised: few rows, of 16 million values each
        _norm("norm_lattices", "norm", "f64", 16, 4096, 4096, affine=False),
        # 64 chains on the 35 x 60 lattice of the tree counts, with a scale and an offset for each site
        _norm("norm_grad_sites", "norm_grad", "f64", 64, 35, 60),
        # four fields on a 1024 x 1024 lattice: rows too few to fill the card by themselves
        _norm("norm_grad_fields", "norm_grad", "f64", 4, 1024, 1024),
        # the class probabilities of one token of a generating model: bound by reading beta once
        _class("class_one_token", "class", "bf16", 1, 4096, 32000),
        # scoring a padded batch: an odd number of classes, a third of the rows behind their sequence's end
        _class("class_tokens", "class", "f16", 2047, 2048, 50001, masked=0.33),
        # one gradient evaluation of a sampler: 8 fields on the 35 x 60 lattice, 300 species, no count at a fifth of the sites
        _class("class_grad_sites", "class_grad", "f64", 2100, 8, 300, masked=0.2),
        # 32 fields on a 256 x 256 lattice
        _class("class_grad_fields", "class_grad", "f32", 65536, 32, 1000, masked=0.1),
        # a training step's loss over a large vocabulary, with its gradients: the largest call
        _class("class_grad_tokens", "class_grad", "bf16", 4096, 4096, 128000, masked=0.05, mean=True),
    ]


def _spread(rng, low, high):
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "class", "class_grad"])
    if op.startswith("norm"):
        dtype = rng.choice(["bf16", "f16", "f32", "f64"])
        affine = rng.random() < 0.75
        if rng.random() < 0.5:  # rows of features
            return _norm(None, op, dtype, _spread(rng, 1, 16384), 1, _spread(rng, 16, 8192), affine)
        rows = _spread(rng, 1, 64)  # lattices
        side = (1 << 26) // rows
        height = _spread(rng, 8, min(4096, side // 8))
        return _norm(None, op, dtype, rows, height, _spread(rng, 8, min(4096, side // height)), affine)
    masked = rng.choice([0.0, 0.1, 0.4, 0.8])
    if rng.random() < 0.5:  # fields on a lattice: many sites, few fields, hundreds of classes
        return _class(None, op, rng.choice(["f64", "f32"]), _spread(rng, 100, 65536), _spread(rng, 1, 64),
                      _spread(rng, 3, 1000), masked)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    top = 1 << (41 if SIZE[dtype] == 2 else 38)
    features = _spread(rng, 64, 4096)
    classes = _spread(rng, 1000, 128000)
    rows = _spread(rng, 1, max(1, min(8192, top // (features * classes))))
    return _class(None, op, dtype, rows, features, classes, masked, mean=dtype == "bf16" and rng.random() < 0.5)


def _wide(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def prepare(case, seed):
    dev = torch.device("cuda")
    rng = torch.Generator(device=dev)
    rng.manual_seed(seed)
    dtype = TYPES[case["type"]]
    wide = _wide(dtype)

    def normal(*shape, scale=1.0, offset=0.0):
        return (torch.randn(shape, generator=rng, device=dev, dtype=wide).mul_(scale).add_(offset)).to(dtype)

    s = {"op": case["op"]}
    if case["op"].startswith("norm"):
        core = (case["width"],) if case["height"] == 1 else (case["height"], case["width"])
        s["core"] = len(core)
        s["x"] = normal(case["rows"], *core, scale=1.7, offset=0.4)
        s["weight"] = normal(*core, scale=0.2, offset=1.0) if case["affine"] else None
        s["bias"] = normal(*core, scale=0.3) if case["affine"] else None
        if case["op"] == "norm_grad":
            s["ybar"] = normal(case["rows"], *core)
            dims = tuple(range(1, 1 + len(core)))
            x = s["x"].to(wide)
            s["mean"] = x.mean(dims)
            var = (x - s["mean"].view(-1, *[1] * len(core))).square_().mean(dims)
            s["rstd"] = (var + EPS).rsqrt()
        return s
    n, d, v = case["rows"], case["features"], case["classes"]
    s["x"] = normal(n, d)
    s["beta"] = normal(v, d, scale=1.5 / d ** 0.5)
    s["alpha"] = normal(v, scale=0.5)
    # some classes are common and most are rare
    y = (torch.rand(n, generator=rng, device=dev, dtype=torch.float64) ** 3 * v).long().clamp_(max=v - 1)
    hidden = int(n * case["masked"])
    if hidden:
        y[torch.randperm(n, generator=rng, device=dev)[:hidden]] = -1
    s["y"] = y
    s["lpbar"] = torch.full((n,), -1.0 / max(1, n - hidden), device=dev, dtype=wide) if case["mean"] else None
    return s


def _plain_norm(s):
    x = s["x"].to(_wide(s["x"].dtype))
    dims = tuple(range(x.ndim - s["core"], x.ndim))
    mean = x.mean(dims, keepdim=True)
    c = x - mean
    rstd = ((c * c).mean(dims, keepdim=True) + EPS).rsqrt()
    y = c * rstd
    if s["weight"] is not None:
        y = y * s["weight"].to(x.dtype) + s["bias"].to(x.dtype)
    return {"y": y.to(s["x"].dtype), "mean": mean.flatten(), "rstd": rstd.flatten()}


def _plain_norm_grad(s):
    x, g = s["x"].to(s["mean"].dtype), s["ybar"].to(s["mean"].dtype)
    dims = tuple(range(x.ndim - s["core"], x.ndim))
    one = [1] * s["core"]
    rstd = s["rstd"].view(-1, *one)
    h = (x - s["mean"].view(-1, *one)) * rstd
    out = {"wbar": (g * h).sum(0).to(s["x"].dtype), "bbar": g.sum(0).to(s["x"].dtype)}
    if s["weight"] is not None:
        g = g * s["weight"].to(g.dtype)
    out["xbar"] = (rstd * (g - g.mean(dims, keepdim=True) - h * (g * h).mean(dims, keepdim=True))).to(s["x"].dtype)
    return out


def _plain_class(s):
    wide = _wide(s["x"].dtype)
    seen = s["y"] >= 0
    x, beta = s["x"].to(wide), s["beta"].to(wide)
    eta = x @ beta.T + s["alpha"].to(wide)
    top = eta.max(1, keepdim=True).values
    e = (eta - top).exp()
    total = e.sum(1, keepdim=True)
    at = s["y"].clamp(min=0).unsqueeze(1)
    lp = (eta.gather(1, at) - top - total.log()).squeeze(1)
    lp = torch.where(seen, lp, torch.zeros_like(lp))
    if s["op"] == "class":
        return {"lp": lp}
    scale = seen.to(wide) if s["lpbar"] is None else torch.where(seen, s["lpbar"], torch.zeros_like(s["lpbar"]))
    r = e.mul_(-scale.unsqueeze(1) / total)
    r.scatter_add_(1, at, scale.unsqueeze(1))
    return {"lp": lp, "xbar": (r @ beta).to(s["x"].dtype), "alphabar": r.sum(0).to(s["x"].dtype),
            "betabar": (r.T @ x).to(s["x"].dtype)}


def run(state):
    s = state
    if own:
        from gptools_amd import glm

        if s["op"] == "norm":
            y, mean, rstd = glm.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, core_ndim=s["core"])
            return {"y": y, "mean": mean, "rstd": rstd}
        if s["op"] == "norm_grad":
            xbar, wbar, bbar = glm.layer_norm_vjp(s["x"], s["weight"], s["mean"], s["rstd"], s["ybar"],
                                                  core_ndim=s["core"])
            return {"wbar": wbar, "bbar": bbar, "xbar": xbar}
        # labels are known to be classes here, as a sampler's or a training loop's are: no check that waits for the GPU
        if s["op"] == "class":
            return {"lp": glm.categorical_logit_glm_lpmf(s["y"], s["x"], s["alpha"], s["beta"], check=False)}
        lp, xbar, alphabar, betabar = glm.categorical_logit_glm_lpmf_vjp(s["y"], s["x"], s["alpha"], s["beta"],
                                                                         lpbar=s["lpbar"], check=False)
        return {"lp": lp, "xbar": xbar, "alphabar": alphabar, "betabar": betabar}
    return {"norm": _plain_norm, "norm_grad": _plain_norm_grad}.get(s["op"], _plain_class)(s)


def work(case):
    b = SIZE[case["type"]]
    wide = 8 if case["type"] == "f64" else 4
    if case["op"].startswith("norm"):
        width = case["height"] * case["width"]
        cells = case["rows"] * width
        params = 2 * width if case["affine"] else 0
        if case["op"] == "norm":
            return {"bytes": b * (2 * cells + params) + 2 * wide * case["rows"], "flops": 8 * cells}
        return {"bytes": b * (3 * cells + params // 2 + 2 * width) + 2 * wide * case["rows"], "flops": 16 * cells}
    n, d, v = case["rows"], case["features"], case["classes"]
    seen = n - int(n * case["masked"])
    inputs = b * (seen * d + v * d + v) + 8 * n
    if case["op"] == "class":
        return {"bytes": inputs + wide * n, "flops": 2 * seen * d * v + 4 * seen * v}
    # three products (logits, xbar, betabar); what a second computation of the logits costs is the kernels' own choice
    return {"bytes": inputs + (wide * n if case["mean"] else 0) + wide * n + b * (n * d + v * d + v),
            "flops": 6 * seen * d * v + 8 * seen * v}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("norm"):
        rows = s["x"].shape[0]
        shape = s["x"].shape
        x = s["x"].reshape(rows, -1)
        w = None if s["weight"] is None else s["weight"].double().flatten()
        ys, gs, means, rstds = [], [], [], []
        wbar = torch.zeros(x.shape[1], dtype=torch.float64, device=x.device)
        bbar = torch.zeros_like(wbar)
        step = max(1, (1 << 27) // x.shape[1])
        for i in range(0, rows, step):
            c = x[i:i + step].double()
            mean = c.sum(1, keepdim=True) / c.shape[1]
            c = c - mean
            rstd = 1.0 / torch.sqrt((c ** 2).sum(1, keepdim=True) / c.shape[1] + EPS)
            h = c * rstd
            means.append(mean.squeeze(1))
            rstds.append(rstd.squeeze(1))
            if case["op"] == "norm":
                ys.append(h if w is None else h * w + s["bias"].double().flatten())
                continue
            g = s["ybar"].reshape(rows, -1)[i:i + step].double()
            wbar += torch.sum(g * h, 0)
            bbar += torch.sum(g, 0)
            if w is not None:
                g = g * w
            gs.append(rstd * (g - g.sum(1, keepdim=True) / g.shape[1] - h * (g * h).sum(1, keepdim=True) / g.shape[1]))
        if case["op"] == "norm":
            return {"y": torch.cat(ys).view(shape), "mean": torch.cat(means), "rstd": torch.cat(rstds)}
        return {"wbar": wbar.view(shape[1:]), "bbar": bbar.view(shape[1:]), "xbar": torch.cat(gs).view(shape)}
    n, d = s["x"].shape
    beta, alpha = s["beta"].double(), s["alpha"].double()
    step = max(1, (1 << 28) // beta.shape[0])
    lp = torch.zeros(n, dtype=torch.float64, device=beta.device)
    xbar = torch.zeros(n, d, dtype=torch.float64, device=beta.device)
    betabar, alphabar = torch.zeros_like(beta), torch.zeros_like(alpha)
    for i in range(0, n, step):
        y = s["y"][i:i + step]
        at = torch.nonzero(y >= 0).squeeze(1)
        if not at.numel():
            continue
        x = s["x"][i:i + step].double()[at]
        logp = torch.mm(x, beta.t()).add_(alpha)
        logp -= logp.amax(1, keepdim=True)
        logp -= torch.log(torch.exp(logp).sum(1, keepdim=True))
        lp[i + at] = logp[torch.arange(len(at), device=at.device), y[at]]
        if case["op"] == "class":
            continue
        r = logp.exp_().neg_()
        r[torch.arange(len(at), device=at.device), y[at]] += 1.0
        if s["lpbar"] is not None:
            r *= s["lpbar"][i + at].double().unsqueeze(1)
        xbar[i + at] = torch.mm(r, beta)
        betabar += torch.mm(r.t().contiguous(), x)
        alphabar += r.sum(0)
    if case["op"] == "class":
        return {"lp": lp}
    return {"lp": lp, "xbar": xbar, "alphabar": alphabar, "betabar": betabar}
