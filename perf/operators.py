"""What is measured of the matrix products that the layers of a language model are made of: products with bias,
activation and residual in their epilogue, their backward pass, and products grouped by expert with ragged sizes.

Five operators, all on row-major matrices in fp32, fp16 or bf16 (sums in 32 bits, one rounding at the end):

  epilogue          Z = A op(B) + bias, C = act(Z) + beta R; Z is kept for the backward pass where `pre` is set
  gradient          dZ = (A op(B)) * act'(Z), db = column sums of dZ: the product that carries a gradient through an activation
  activation        dZ = dY * act'(Z), db_g = column sums of dZ over the rows of group g: the same without a product
  grouped           for the rows of group g: Z = A_g op(B_g) + bias_g, C = act(Z): the experts' products
  grouped_gradient  C_g = A_g^T B_g: the gradients of the experts' weights

The groups are given by `offsets` on the GPU (group g owns the rows offsets[g] .. offsets[g + 1] - 1), as a router leaves
them there; rows behind the last group belong to nobody and are left as they were.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token of a conversation through the first layer of a feed-forward block: bound by reading the weights once
        {"name": "epilogue, one token", "op": "epilogue", "type": "bf16", "m": 1, "n": 8192, "k": 4096, "transposed": True,
         "act": "gelu", "bias": True, "pre": False, "residual": False, "pad": 0},
        # a prompt (or a training batch) of 8192 tokens through the same layer, the activation's input kept for training
        {"name": "epilogue, prompt", "op": "epilogue", "type": "bf16", "m": 8192, "n": 8192, "k": 4096, "transposed": True,
         "act": "gelu", "bias": True, "pre": True, "residual": False, "pad": 0},
        # a head of odd width behind a layer of odd width: no row starts at an aligned address
        {"name": "epilogue, odd sizes", "op": "epilogue", "type": "fp16", "m": 777, "n": 1001, "k": 1023, "transposed": True,
         "act": "silu", "bias": True, "pre": False, "residual": True, "pad": 0},
        # the second layer of a feed-forward block trained in 32 bits, with the residual stream added
        {"name": "epilogue, fp32", "op": "epilogue", "type": "fp32", "m": 1024, "n": 1024, "k": 4096, "transposed": False,
         "act": "none", "bias": True, "pre": False, "residual": True, "pad": 0},
        # backward pass of a feed-forward block: the gradient of its second product, through the activation, and the bias's
        {"name": "gradient, batch", "op": "gradient", "type": "bf16", "m": 4096, "n": 8192, "k": 2048, "transposed": False,
         "act": "gelu", "pad": 0},
        # the same for a small model in 32 bits
        {"name": "gradient, small fp32", "op": "gradient", "type": "fp32", "m": 300, "n": 1000, "k": 512, "transposed": False,
         "act": "silu", "pad": 0},
        # the activation's backward pass where the gradient comes from elsewhere: one pass over three large matrices
        {"name": "activation, batch", "op": "activation", "type": "bf16", "rows": 8192, "n": 8192, "groups": 1, "act": "gelu", "pad": 0},
        # the same behind experts, with one bias gradient for each of them
        {"name": "activation, by expert", "op": "activation", "type": "fp16", "rows": 4099, "n": 1024, "groups": 32, "act": "silu", "pad": 0},
        # a step of serving: 16 tokens, eight experts of 64 each; bound by reading the chosen experts' weights
        {"name": "grouped, serving", "op": "grouped", "type": "bf16", "rows": 128, "n": 2048, "k": 1024, "groups": 64,
         "transposed": True, "act": "silu", "bias": False, "pre": False, "pad": 0},
        # a prompt or a training batch: 16384 rows over 16 experts, unevenly
        {"name": "grouped, batch", "op": "grouped", "type": "bf16", "rows": 16384, "n": 4096, "k": 2048, "groups": 16,
         "transposed": False, "act": "silu", "bias": True, "pre": True, "pad": 0},
        # the gradients of those experts' weights
        {"name": "grouped gradient, batch", "op": "grouped_gradient", "type": "bf16", "rows": 16384, "m": 2048, "n": 4096, "groups": 16, "pad": 0},
        # a small step of many small experts, some of them without a row
        {"name": "grouped gradient, small", "op": "grouped_gradient", "type": "fp16", "rows": 1501, "m": 520, "n": 1000, "groups": 24, "pad": 0},
    ]


def draw(rng):
    def size(low, high):  # spread over the logarithm; one in six of any value, the others multiples of 8 where large enough
        v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        if v >= 64 and rng.random() > 1 / 6:
            v = (v + 4) // 8 * 8
        return max(low, min(high, v))

    op = rng.choice(["epilogue", "epilogue", "gradient", "activation", "grouped", "grouped", "grouped_gradient"])
    kind = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
    most = 1.5e11 if kind == "fp32" else 5e11  # operations: no drawn case costs more than the largest listed ones
    case = {"op": op, "type": kind, "pad": rng.choice([0, 0, 8, 24, 1])}
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    while True:
        if op in ("epilogue", "gradient"):
            m, n, k = size(1, 8192), size(64, 8192), size(64, 8192)
            if 2 * m * n * k <= most:
                break
        elif op == "activation":
            m, n, k = size(1, 8192), size(64, 8192), 0
            break
        elif op == "grouped":
            m, n, k, g = size(1, 16384), size(64, 4096), size(64, 4096), size(1, 64)
            if 2 * m * n * k <= most and g * n * k <= 1 << 28:
                break
        else:
            m, n, k, g = size(64, 4096), size(64, 4096), size(1, 16384), size(1, 64)
            if 2 * m * n * k <= most and g * n * m <= 1 << 28:
                break
    if op == "epilogue":
        case.update(m=m, n=n, k=k, transposed=rng.random() < 0.5, act=act, bias=rng.random() < 0.7, pre=rng.random() < 0.3,
                    residual=rng.random() < 0.4)
    elif op == "gradient":
        case.update(m=m, n=n, k=k, transposed=rng.random() < 0.5, act=act)
    elif op == "activation":
        case.update(rows=m, n=n, groups=rng.choice([1, 1, size(2, 64)]), act=act)
    elif op == "grouped":
        case.update(rows=m, n=n, k=k, groups=g, transposed=rng.random() < 0.5, act=act, bias=rng.random() < 0.5, pre=rng.random() < 0.3)
    else:
        case.update(rows=k, m=m, n=n, groups=g)
    return case


def _sizes(rows, groups, seed):
    """Rows of each group: a router's uneven choice; about one row in fifty belongs to nobody (the padding of a batch)."""
    r = np.random.RandomState(seed % (1 << 31))
    if groups == 1:
        return [rows - rows // 50]
    return [int(v) for v in r.multinomial(rows - rows // 50, r.dirichlet(np.full(groups, 2.0)))]


def prepare(case, seed):
    dtype, op, pad = _TYPES[case["type"]], case["op"], case["pad"]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def matrix(rows, cols, scale=1.0):  # `pad` more elements from row to row than a row has
        v = torch.randn(rows, cols + pad, generator=g, device="cuda") * scale
        return v.to(dtype)[:, :cols]

    def empty(rows, cols):
        return torch.zeros(rows, cols + pad, device="cuda", dtype=dtype)[:, :cols]

    s = {"case": case}
    if "groups" in case:
        s["sizes"] = _sizes(case["rows"], case["groups"], seed)
        s["offsets"] = torch.tensor(np.concatenate([[0], np.cumsum(s["sizes"])]), dtype=torch.int64, device="cuda")
    if op in ("epilogue", "gradient"):
        m, n, k = case["m"], case["n"], case["k"]
        s["a"] = matrix(m, k)
        s["b"] = matrix(n, k, k ** -0.5) if case["transposed"] else matrix(k, n, k ** -0.5)
        s["c"] = empty(m, n)
        if op == "gradient":
            s["pre"] = matrix(m, n)
            s["db"] = torch.zeros(n, device="cuda", dtype=dtype)
        else:
            s["bias"] = matrix(1, n, 0.1)[0] if case["bias"] else None
            s["residual"] = matrix(m, n) if case["residual"] else None
            s["pre"] = empty(m, n) if case["pre"] else None
    elif op == "activation":
        rows, n = case["rows"], case["n"]
        s["a"], s["pre"], s["c"] = matrix(rows, n), matrix(rows, n), empty(rows, n)
        s["db"] = torch.zeros(case["groups"], n, device="cuda", dtype=dtype)
    elif op == "grouped":
        rows, n, k, groups = case["rows"], case["n"], case["k"], case["groups"]
        s["a"] = matrix(rows, k)
        shape = (groups, n, k) if case["transposed"] else (groups, k, n)
        s["b"] = (torch.randn(shape, generator=g, device="cuda") * k ** -0.5).to(dtype)
        s["bias"] = (torch.randn(groups, n, generator=g, device="cuda") * 0.1).to(dtype) if case["bias"] else None
        s["c"] = empty(rows, n)
        s["pre"] = empty(rows, n) if case["pre"] else None
    else:
        rows, m, n, groups = case["rows"], case["m"], case["n"], case["groups"]
        s["a"], s["b"] = matrix(rows, m), matrix(rows, n)
        s["c"] = torch.zeros(groups, m, n, device="cuda", dtype=dtype)
    return s


# ---- the plain forms: elementary operations in 32 bits, one rounding at the end -----------------------------------------

def _act(z, kind):
    if kind == "relu":
        return torch.clamp(z, min=0)
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z / (1 + torch.exp(-z)) if kind == "silu" else z


def _slope(z, kind):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if kind == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _product(a, b, transposed):
    b = b.float()
    return a.float() @ (b.T if transposed else b)


def _plain(s):
    c = s["case"]
    op, dtype = c["op"], s["a"].dtype
    if op == "epilogue":
        z = _product(s["a"], s["b"], c["transposed"])
        if c["bias"]:
            z = z + s["bias"].float()
        y = _act(z, c["act"])
        if c["residual"]:
            y = y + s["residual"].float()
        return {"c": y.to(dtype), "pre": z.to(dtype)} if c["pre"] else {"c": y.to(dtype)}
    if op == "gradient":
        dz = _product(s["a"], s["b"], c["transposed"]) * _slope(s["pre"].float(), c["act"])
        return {"c": dz.to(dtype), "db": dz.sum(0).to(dtype)}
    # The groups one after the other, as programs without a grouped product do it; the host knows their sizes here, which
    # spares this form the wait for the router's counts.
    at, sums, here = 0, [], slice(0, sum(s["sizes"]))
    out = {k: torch.zeros(s[k].shape, dtype=dtype, device="cuda") for k in ("c", "pre") if s.get(k) is not None and (k == "c" or op == "grouped")}
    if op == "activation":
        dz = s["a"][here].float() * _slope(s["pre"][here].float(), c["act"])
        out["c"][here] = dz.to(dtype)
    for g, rows in enumerate(s["sizes"]):
        here = slice(at, at + rows)
        at += rows
        if op == "activation":
            sums.append(dz[here].sum(0))
        elif op == "grouped" and rows:
            z = _product(s["a"][here], s["b"][g], c["transposed"])
            if c["bias"]:
                z = z + s["bias"][g].float()
            if c["pre"]:
                out["pre"][here] = z.to(dtype)
            out["c"][here] = _act(z, c["act"]).to(dtype)
        elif op == "grouped_gradient" and rows:
            out["c"][g] = (s["a"][here].float().T @ s["b"][here].float()).to(dtype)
    if sums:
        out["db"] = torch.stack(sums).to(dtype)
    return out


# ---- the framework's calls --------------------------------------------------------------------------------------------

def _calls(s):
    from clblast_amd import api
    c, a, out = s["case"], s["a"], s["c"]
    op = c["op"]
    if op == "epilogue":
        pre, residual = s["pre"], s["residual"]
        api.gemmEpilogue(None, c["m"], c["n"], c["k"], a, s["b"], out, a.stride(0), s["b"].stride(0), out.stride(0),
                         b_transp=c["transposed"], activation=c["act"], bias=s["bias"], pre=pre,
                         pre_ld=0 if pre is None else pre.stride(0), beta=0.0 if residual is None else 1.0, residual=residual,
                         residual_ld=0 if residual is None else residual.stride(0))
        return {"c": out, "pre": pre} if c["pre"] else {"c": out}
    if op == "gradient":
        api.gemmActivationGradient(None, c["m"], c["n"], c["k"], a, s["b"], s["pre"], out, a.stride(0), s["b"].stride(0),
                                   s["pre"].stride(0), out.stride(0), b_transp=c["transposed"], activation=c["act"],
                                   bias_gradient=s["db"])
        return {"c": out, "db": s["db"]}
    if op == "activation":
        api.activationGradient(None, c["rows"], c["n"], a, s["pre"], out, a.stride(0), s["pre"].stride(0), out.stride(0),
                               activation=c["act"], bias_gradient=s["db"], group_count=c["groups"], group_offsets=s["offsets"])
        return {"c": out, "db": s["db"]}
    if op == "grouped":
        pre = s["pre"]
        api.gemmGrouped(None, c["groups"], c["rows"], c["n"], c["k"], a, s["b"], out, s["offsets"], a.stride(0), s["b"].stride(1),
                        out.stride(0), b_stride=s["b"].stride(0), b_transp=c["transposed"], activation=c["act"], bias=s["bias"],
                        pre=pre, pre_ld=0 if pre is None else pre.stride(0))
        return {"c": out, "pre": pre} if c["pre"] else {"c": out}
    api.gemmGroupedGradient(None, c["groups"], c["rows"], c["m"], c["n"], a, s["b"], out, s["offsets"], a.stride(0),
                            s["b"].stride(0), out.stride(1), c_stride=out.stride(0))
    return {"c": out}


def run(state):
    return _calls(state) if own else _plain(state)


def work(case):
    size, op, n = 4 if case["type"] == "fp32" else 2, case["op"], case["n"]
    if op in ("epilogue", "gradient"):
        m, k = case["m"], case["k"]
        matrices = 2 if op == "gradient" else 1 + case["pre"] + case["residual"]
        values = m * k + k * n + matrices * m * n + (n if op == "gradient" or case["bias"] else 0)
        return {"bytes": size * values, "flops": 2 * m * n * k}
    rows, groups = case["rows"] - case["rows"] // 50, case["groups"]
    if op == "activation":
        return {"bytes": size * (3 * rows * n + groups * n), "flops": 20 * rows * n}
    # the weights of experts without a row are not read: the mean number of the others
    used = sum(sum(v > 0 for v in _sizes(case["rows"], groups, seed)) for seed in range(8)) / 8
    if op == "grouped":
        k = case["k"]
        return {"bytes": size * (rows * k + used * (n * k + (n if case["bias"] else 0)) + (1 + case["pre"]) * rows * n), "flops": 2 * rows * n * k}
    m = case["m"]
    return {"bytes": size * (rows * (m + n) + groups * m * n), "flops": 2 * rows * m * n}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    wide = {k: v.double() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}

    def phi(z):  # the normal distribution function
        return torch.special.erfc(-z / math.sqrt(2)) / 2

    def inner(z):
        return math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)

    value = {"none": lambda z: z, "relu": lambda z: torch.where(z > 0, z, 0.0), "gelu": lambda z: z * phi(z),
             "gelu_tanh": lambda z: z * torch.sigmoid(2 * inner(z)), "silu": lambda z: z * torch.sigmoid(z)}
    slope = {"none": lambda z: torch.ones_like(z), "relu": lambda z: torch.where(z > 0, 1.0, 0.0).double(),
             "gelu": lambda z: phi(z) + z * torch.exp(-z ** 2 / 2) / math.sqrt(2 * math.pi),
             "gelu_tanh": lambda z: torch.sigmoid(2 * inner(z)) + z * torch.sigmoid(2 * inner(z)) * torch.sigmoid(-2 * inner(z))
             * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z ** 2),
             "silu": lambda z: torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)}
    op, act, n = case["op"], case.get("act", "none"), case["n"]
    if op in ("epilogue", "gradient"):
        z = torch.mm(wide["a"], wide["b"].t() if case["transposed"] else wide["b"])
        if op == "gradient":
            dz = torch.mul(z, slope[act](wide["pre"]))
            return {"c": dz, "db": torch.mv(dz.t(), torch.ones(case["m"], dtype=torch.float64, device="cuda"))}
        if case["bias"]:
            z += wide["bias"]
        y = value[act](z)
        if case["residual"]:
            y = torch.add(wide["residual"], y)
        return {"c": y, "pre": z} if case["pre"] else {"c": y}
    rows, groups = case["rows"], case["groups"]
    ends = s["offsets"].tolist()
    owner = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    for g in range(groups):
        owner[ends[g]:ends[g + 1]] = g
    if op == "activation":
        dz = wide["a"] * slope[act](wide["pre"]) * (owner >= 0)[:, None]
        db = torch.zeros(groups, n, dtype=torch.float64, device="cuda").index_add_(0, owner.clamp(min=0), dz)
        return {"c": dz, "db": db}
    if op == "grouped":
        y, z = (torch.zeros(rows, n, dtype=torch.float64, device="cuda") for _ in range(2))
        for g in range(groups):
            mine = (owner == g).nonzero()[:, 0]
            w = wide["b"][g]
            zg = torch.mm(wide["a"][mine], w.t() if case["transposed"] else w)
            zg = zg + wide["bias"][g] if case["bias"] else zg
            y[mine], z[mine] = value[act](zg), zg
        return {"c": y, "pre": z} if case["pre"] else {"c": y}
    c = torch.zeros(groups, case["m"], n, dtype=torch.float64, device="cuda")
    for g in range(groups):
        mine = (owner == g).nonzero()[:, 0]
        c[g] = torch.mm(wide["a"][mine].t(), wide["b"][mine])
    return {"c": c}
