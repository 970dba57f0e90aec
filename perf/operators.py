"""What is measured of the block's dense layers, group norm and dropout.

The operators are those around the selective scan in a BidirectionalMamba block
(norm, projections and the MLP with its dropout):

* ``group_norm_act``  activation(group norm of channels-last x)
* ``dropout_act``     residual + activation(dropout(x)), mask from a counter-based generator
* ``dense_act``       residual + activation(dropout(x @ kernel + bias))

``run`` computes them with elementary torch operations in 32 bits (``own`` false) or with the package's
operators (``own`` true); ``exact`` gives the definition in 64 bits.

Dropout's random bits are Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
1, 2, 3", 2011).  With ``rng = (seed, offset)`` the element in column c of row r (rows of the last axis, of C
columns) takes the 16 bits number c % 8 of the 128 bits of counter (r * ceil(C / 8) + c // 8, offset) under
the key seed, and is kept if they are at least ``round(rate * 65536)``.
"""

import math

import numpy as np
import torch

own = False

GELU_C = 0.7978845608028654  # sqrt(2 / pi)


def listed():
    return [
        # one sequence, one new token through the first MLP layer while generating: latency
        {"name": "dense-token", "op": "dense", "rows": 1, "fin": 768, "fout": 1536, "dtype": "bf16", "act": "silu",
         "residual": False, "rate": 0.0, "train": False},
        # a token each of a few sequences through an fp32 model's second MLP layer, residual added: latency
        {"name": "dense-few-tokens-fp32", "op": "dense", "rows": 12, "fin": 1024, "fout": 512, "dtype": "fp32",
         "act": None, "residual": True, "rate": 0.0, "train": False},
        # a training step of an fp32 model with sizes that fit no tile and rows that start at no 16-byte boundary
        {"name": "dense-odd-fp32-train", "op": "dense", "rows": 2042, "fin": 515, "fout": 1001, "dtype": "fp32",
         "act": "gelu", "residual": False, "rate": 0.2, "train": True},
        # a training step of the first MLP layer, 16 sequences of 2048: products in all three directions
        {"name": "dense-up-train", "op": "dense", "rows": 32768, "fin": 768, "fout": 1536, "dtype": "bf16",
         "act": "silu", "residual": False, "rate": 0.1, "train": True},
        # the second MLP layer over the whole batch of 64 sequences of 2048, dropout and residual, forward
        {"name": "dense-down-batch", "op": "dense", "rows": 131072, "fin": 1536, "fout": 768, "dtype": "bf16",
         "act": None, "residual": True, "rate": 0.1, "train": False},
        # one token of each of 64 sequences through the block's norm: latency
        {"name": "norm-tokens", "op": "norm", "batch": 64, "length": 1, "dim": 768, "groups": 32, "dtype": "bf16",
         "act": "silu", "train": False},
        # a training step with a ragged length, few sequences and groups of an odd width
        {"name": "norm-odd-fp32-train", "op": "norm", "batch": 3, "length": 1021, "dim": 330, "groups": 10,
         "dtype": "fp32", "act": "gelu", "train": True},
        # the norm of the whole batch, forward
        {"name": "norm-batch", "op": "norm", "batch": 64, "length": 2048, "dim": 768, "groups": 32, "dtype": "bf16",
         "act": None, "train": False},
        # a training step on two long DNA sequences: few rows of statistics, each over a million values
        {"name": "norm-long-train", "op": "norm", "batch": 2, "length": 131072, "dim": 256, "groups": 32,
         "dtype": "bf16", "act": "silu", "train": True},
        # dropout and activation of one small fp32 batch: latency
        {"name": "dropout-small", "op": "dropout", "rows": 2048, "dim": 128, "dtype": "fp32", "act": "silu",
         "residual": False, "rate": 0.1, "train": False},
        # ragged rows of an odd width with a residual
        {"name": "dropout-odd-train", "op": "dropout", "rows": 5005, "dim": 333, "dtype": "fp32", "act": "relu",
         "residual": True, "rate": 0.25, "train": True},
        # a training step of the MLP's hidden layer over the batch of 64 sequences of 2048
        {"name": "dropout-batch-train", "op": "dropout", "rows": 131072, "dim": 768, "dtype": "bf16", "act": "silu",
         "residual": False, "rate": 0.1, "train": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: any integer for a third of the draws, otherwise a multiple of 8."""
    n = _log_int(rng, lo, hi)
    n = n if rng.random() < 0.34 else max(8, n // 8 * 8)
    return n + 8 if n == 2 * 1536 else n


def draw(rng):
    op = rng.choice(["dense", "dense", "norm", "dropout"])
    case = {"op": op, "dtype": rng.choice(["fp32", "bf16"]), "act": rng.choice([None, "silu", "gelu", "relu"]),
            "train": rng.random() < 0.5}
    if op == "dense":
        case["fin"], case["fout"] = _width(rng, 32, 2048), _width(rng, 32, 2048)
        most = 2.0e10 if case["dtype"] == "fp32" else 1.0e11
        most = min(most / (2.0 * case["fin"] * case["fout"]) / (3 if case["train"] else 1), 65536)
        case["rows"] = _log_int(rng, 1, max(most, 2))
        case["residual"] = rng.random() < 0.5
        case["rate"] = rng.choice([0.0, round(rng.uniform(0.05, 0.6), 3)])
    elif op == "norm":
        case["groups"] = rng.choice([1, 4, 8, 15, 32, 32, 32])
        case["dim"] = case["groups"] * _log_int(rng, 1 if case["groups"] > 8 else 8, 2048 // case["groups"])
        case["batch"] = _log_int(rng, 1, 64)
        case["length"] = _log_int(rng, 1, max(2, 5.0e7 / case["dim"] / case["batch"]))
    else:
        case["dim"] = _width(rng, 8, 2048)
        case["rows"] = _log_int(rng, 1, 5.0e7 / case["dim"])
        case["residual"] = rng.random() < 0.5
        case["rate"] = round(rng.uniform(0.02, 0.7), 3)
    return case


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = {"fp32": torch.float32, "bf16": torch.bfloat16}[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0, dtype=dt):
        return (mean + scale * torch.randn(*shape, device="cuda", generator=g)).to(dtype)

    st = {"case": case, "rng": (1_000_003 * (seed + 1), 17 + seed)}
    if case["op"] == "dense":
        m, k, n = case["rows"], case["fin"], case["fout"]
        st["x"] = normal(m, k)
        st["kernel"] = normal(k, n, scale=k ** -0.5)
        st["bias"] = normal(n, scale=0.1)
        if case["residual"]:
            st["residual"] = normal(m, n)
        if case["train"]:
            st["dy"] = normal(m, n)
    elif case["op"] == "norm":
        b, l, d = case["batch"], case["length"], case["dim"]
        offset = normal(d, scale=0.5, dtype=torch.float32)
        st["x"] = (offset + normal(b, l, d, dtype=torch.float32)).to(dt)
        st["scale"] = normal(d, scale=0.1, mean=1.0, dtype=torch.float32)
        st["bias"] = normal(d, scale=0.1, dtype=torch.float32)
        if case["train"]:
            st["dy"] = normal(b, l, d)
    else:
        m, d = case["rows"], case["dim"]
        st["x"] = normal(m, d)
        if case["residual"]:
            st["residual"] = normal(m, d)
        if case["train"]:
            st["dy"] = normal(m, d)
    if case["train"]:
        for name in ("x", "kernel", "scale", "bias"):
            if name in st:
                st[name].requires_grad_()
    return st


# ----------------------------------------------------------------------------- the package's operators
def _run_own(st):
    import selectssm_b200 as S
    case = st["case"]
    if case["op"] == "dense":
        y = S.dense_act(st["x"], st["kernel"], st["bias"], activation=case["act"], residual=st.get("residual"),
                        rate=case["rate"], rng=st["rng"])
        leaves = ("x", "kernel", "bias")
    elif case["op"] == "norm":
        y = S.group_norm_act(st["x"], st["scale"], st["bias"], groups=case["groups"], activation=case["act"])
        leaves = ("x", "scale", "bias")
    else:
        y = S.dropout_act(st["x"], case["rate"], st["rng"], activation=case["act"], residual=st.get("residual"))
        leaves = ("x",)
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [st[n] for n in leaves], st["dy"])
    return {"y": y.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}


# ----------------------------------------------------------------------------- the plain form, 32 bits
def _act(u, act):
    if act == "silu":
        return u / (1 + torch.exp(-u))
    if act == "gelu":
        return 0.5 * u * (1 + torch.tanh(GELU_C * (u + 0.044715 * u * u * u)))
    if act == "relu":
        return torch.where(u > 0, u, torch.zeros_like(u))
    return u


def _act_grad(u, act):
    if act == "silu":
        s = 1 / (1 + torch.exp(-u))
        return s * (1 + u * (1 - s))
    if act == "gelu":
        t = torch.tanh(GELU_C * (u + 0.044715 * u * u * u))
        return 0.5 * (1 + t) + 0.5 * u * (1 - t * t) * GELU_C * (1 + 3 * 0.044715 * u * u)
    if act == "relu":
        return (u > 0).to(u.dtype)
    return torch.ones_like(u)


def _keep(rows, cols, rate, rng, device):
    """The (rows, cols) boolean mask, in 64-bit integer operations."""
    seed, offset = rng
    low = 0xFFFFFFFF
    blocks = -(-cols // 8)
    n = torch.arange(rows * blocks, device=device)
    c0, c1 = n & low, n >> 32
    c2, c3 = torch.full_like(n, offset & low), torch.full_like(n, (offset >> 32) & low)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64-bit products; the high half of a wrapped one is masked out
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], dim=1)
    bits = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(rows, blocks * 8)[:, :cols]
    return bits >= round(rate * 65536)


def _drop(u, rate, keep):
    if keep is None:
        return u
    kept = 65536 - round(rate * 65536)
    return torch.where(keep, u * (65536.0 / kept), torch.zeros_like(u))


@torch.no_grad()
def _run_plain(st):
    case, dt = st["case"], st["x"].dtype
    x = st["x"].float()
    act, train = case["act"], case["train"]
    if case["op"] == "norm":
        b, l, d = x.shape
        groups = case["groups"]
        xg = x.reshape(b, l, groups, d // groups)
        mean = xg.mean(dim=(1, 3), keepdim=True)
        xc = xg - mean
        rstd = 1 / torch.sqrt((xc * xc).mean(dim=(1, 3), keepdim=True) + 1e-6)
        xhat = (xc * rstd).reshape(b, l, d)
        u = xhat * st["scale"] + st["bias"]
        out = {"y": _act(u, act).to(dt)}
        if train:
            du = st["dy"].float() * _act_grad(u, act)
            out["dscale"], out["dbias"] = (du * xhat).sum(dim=(0, 1)), du.sum(dim=(0, 1))
            gg, hg = (du * st["scale"]).reshape(xg.shape), xhat.reshape(xg.shape)
            dx = rstd * (gg - gg.mean(dim=(1, 3), keepdim=True) - hg * (gg * hg).mean(dim=(1, 3), keepdim=True))
            out["dx"] = dx.reshape(b, l, d).to(dt)
        return out
    if case["op"] == "dense":
        pre = x @ st["kernel"].float() + st["bias"].float()
    else:
        pre = x
    keep = _keep(pre.shape[0], pre.shape[1], case["rate"], st["rng"], x.device) if case["rate"] > 0 else None
    u = _drop(pre, case["rate"], keep)
    y = _act(u, act)
    if "residual" in st:
        y = y + st["residual"].float()
    out = {"y": y.to(dt)}
    if train:
        dpre = _drop(st["dy"].float() * _act_grad(u, act), case["rate"], keep)
        if case["op"] == "dense":
            out["dx"] = (dpre @ st["kernel"].float().T).to(dt)
            out["dkernel"] = (x.T @ dpre).to(dt)
            out["dbias"] = dpre.sum(dim=0).to(dt)
        else:
            out["dx"] = dpre.to(dt)
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------------------------------- work
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    train = case["train"]
    if case["op"] == "dense":
        m, k, n = case["rows"], case["fin"], case["fout"]
        elems = m * k + k * n + n + m * n + (m * n if case["residual"] else 0)  # x, kernel, bias, y, residual
        if train:
            elems += m * n + m * k + k * n + n  # dy, dx, dkernel, dbias
        return {"bytes": size * elems, "flops": (3 if train else 1) * 2 * m * n * k}
    if case["op"] == "norm":
        n, d = case["batch"] * case["length"] * case["dim"], case["dim"]
        # x, y (dy, dx); scale and bias (and their gradients) in 32 bits
        return {"bytes": (4 if train else 2) * size * n + (4 if train else 2) * 4 * d, "flops": (20 if train else 8) * n}
    n = case["rows"] * case["dim"]
    # x, y, the residual, dy, dx
    return {"bytes": size * n * (2 + (1 if case["residual"] else 0) + (2 if train else 0)),
            "flops": (12 if train else 6) * n}


# ----------------------------------------------------------------------------- the definition in 64 bits
def _philox_keep(rows, cols, rate, rng):
    """The mask again, in numpy's unsigned integers, block of counters by block of counters."""
    threshold = int(round(rate * 65536))
    per_row = (cols + 7) // 8
    out = np.empty((rows * per_row, 8), dtype=np.bool_)
    mult = (np.uint64(0xD2511F53), np.uint64(0xCD9E8D57))
    mask, half = np.uint64(2 ** 32 - 1), np.uint64(32)
    for first in range(0, rows * per_row, 1 << 18):
        count = np.arange(first, min(first + (1 << 18), rows * per_row), dtype=np.uint64)
        ctr = [count & mask, count >> half, np.full_like(count, rng[1] % 2 ** 32),
               np.full_like(count, (rng[1] >> 32) % 2 ** 32)]
        key = [rng[0] % 2 ** 32, (rng[0] >> 32) % 2 ** 32]
        for _ in range(10):
            a, b = mult[0] * ctr[0], mult[1] * ctr[2]
            ctr = [(b >> half) ^ ctr[1] ^ np.uint64(key[0]), b & mask, (a >> half) ^ ctr[3] ^ np.uint64(key[1]), a & mask]
            key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
        block = out[first:first + len(count)]
        for j in range(8):
            block[:, j] = ((ctr[j // 2] >> np.uint64(16 * (j % 2))) & np.uint64(0xFFFF)) >= threshold
    return out.reshape(rows, per_row * 8)[:, :cols]


def _value_and_slope(u, act):
    """activation(u) and its derivative in 64 bits, from the logistic function and tanh's exponential form."""
    if act == "silu":
        sig = torch.where(u >= 0, 1 / (1 + torch.exp(-u.abs())), torch.exp(-u.abs()) / (1 + torch.exp(-u.abs())))
        return u * sig, sig + u * sig * (1 - sig)
    if act == "gelu":
        inner = 2 * math.sqrt(2 / math.pi) * (u + 0.044715 * u ** 3)
        phi = 1 / (1 + torch.exp(-inner))  # (1 + tanh(inner / 2)) / 2
        return u * phi, phi + u * phi * (1 - phi) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * u ** 2)
    if act == "relu":
        return u.clamp(min=0), torch.sign(u).clamp(min=0)
    return u, torch.ones_like(u)


@torch.no_grad()
def exact(case, seed):
    st = {k: v.detach().double() if torch.is_tensor(v) else v for k, v in prepare(case, seed).items()}
    x, act = st["x"], case["act"]
    if case["op"] == "norm":
        b, l, d = x.shape
        rows = x.view(b, l, case["groups"], -1).transpose(1, 2).reshape(b, case["groups"], -1)
        count = rows.shape[2]
        mu = rows.sum(2, keepdim=True) / count
        sd = torch.sqrt(((rows - mu) ** 2).sum(2, keepdim=True) / count + 1e-6)

        def back(t):  # (b, groups, l * width) -> (b, l, d)
            return t.view(b, case["groups"], l, -1).transpose(1, 2).reshape(b, l, d)

        def forth(t):
            return t.view(b, l, case["groups"], -1).transpose(1, 2).reshape(b, case["groups"], -1)

        z = (rows - mu) / sd
        value, slope = _value_and_slope(back(z) * st["scale"] + st["bias"], act)
        out = {"y": value}
        if case["train"]:
            du = st["dy"] * slope
            out["dscale"], out["dbias"] = (du * back(z)).sum((0, 1)), du.sum((0, 1))
            gz = forth(du * st["scale"])
            out["dx"] = back((gz - gz.sum(2, keepdim=True) / count - z * (gz * z).sum(2, keepdim=True) / count) / sd)
        return out
    pre = torch.addmm(st["bias"], x, st["kernel"]) if case["op"] == "dense" else x
    if case["rate"] > 0:
        keep = torch.from_numpy(np.ascontiguousarray(_philox_keep(pre.shape[0], pre.shape[1], case["rate"], st["rng"])))
        factor = keep.to(x.device).double() * (65536 / (65536 - round(case["rate"] * 65536)))
    else:
        factor = torch.ones((), dtype=torch.float64, device=x.device)
    value, slope = _value_and_slope(pre * factor, act)
    out = {"y": value + st["residual"] if "residual" in st else value}
    if case["train"]:
        dpre = st["dy"] * slope * factor
        if case["op"] == "dense":
            out.update(dx=dpre @ st["kernel"].t(), dkernel=(dpre.t() @ x).t(), dbias=dpre.sum(0))
        else:
            out["dx"] = dpre
    return out
