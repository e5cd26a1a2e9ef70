"""Workloads of the transformer operators: attention over the atoms of each structure with its first and second
derivatives, dropout from a counter-based generator, and the lookup of element rows with its gradient.

``run`` computes each in its plain form (elementary torch operations over padded structures), or, where ``own`` is set,
through the package's entry points.
"""
from __future__ import annotations

import functools
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "float64": torch.float64}

ATTENTION = ("attention", "attention_train", "attention_force_train")


def listed():
    return [
        # one molecule of an MD run with a one-head model of the default width: latency only
        {"name": "attention_one_molecule", "kind": "attention", "structures": 1, "lo": 21, "hi": 21, "heads": 1,
         "kv_heads": 1, "dim": 64, "dtype": "float32", "masked": 0.0, "tail": 0},
        # one large simulation box evaluated with eight heads
        {"name": "attention_box", "kind": "attention", "structures": 1, "lo": 8000, "hi": 8000, "heads": 8,
         "kv_heads": 8, "dim": 64, "dtype": "float32", "masked": 0.0, "tail": 0},
        # a double-precision check run over small molecules, odd head width, heads that share keys
        {"name": "attention_train_double", "kind": "attention_train", "structures": 24, "lo": 3, "hi": 29, "heads": 4,
         "kv_heads": 2, "dim": 20, "dtype": "float64", "masked": 0.0, "tail": 0},
        # a training batch of small organic molecules (QM9's sizes), one head
        {"name": "attention_train_molecules", "kind": "attention_train", "structures": 512, "lo": 9, "hi": 29,
         "heads": 1, "kv_heads": 1, "dim": 64, "dtype": "float32", "masked": 0.0, "tail": 0},
        # a padded training batch of drug-sized molecules and peptides at the widest head
        {"name": "attention_train_peptides", "kind": "attention_train", "structures": 40, "lo": 40, "hi": 220,
         "heads": 4, "kv_heads": 4, "dim": 128, "dtype": "float32", "masked": 0.0, "tail": 37},
        # a few proteins or cells, heads that share keys, some atoms (ghosts) that nobody attends to
        {"name": "attention_train_proteins", "kind": "attention_train", "structures": 4, "lo": 1500, "hi": 2500,
         "heads": 8, "kv_heads": 2, "dim": 64, "dtype": "float32", "masked": 0.05, "tail": 0},
        # force training: the forces are a first derivative, the loss takes a second one
        {"name": "force_train_molecules", "kind": "attention_force_train", "structures": 64, "lo": 20, "hi": 70,
         "heads": 1, "kv_heads": 1, "dim": 64, "dtype": "float32", "masked": 0.0, "tail": 0},
        {"name": "force_train_cells", "kind": "attention_force_train", "structures": 2, "lo": 700, "hi": 1000,
         "heads": 4, "kv_heads": 4, "dim": 32, "dtype": "float32", "masked": 0.0, "tail": 0},
        # dropout of attention weights: edges x heads of a small batch
        {"name": "dropout_edges", "kind": "dropout", "rows": 1201, "shared": 1, "inner": 8, "p": 0.1,
         "dtype": "float32"},
        # dropout of equivariant features: one mask for all 49 coefficients (l <= 6) of a node's channel
        {"name": "dropout_coefficients", "kind": "dropout", "rows": 8000, "shared": 49, "inner": 128, "p": 0.2,
         "dtype": "float32"},
        # element rows of a small batch's atoms
        {"name": "embedding_atoms", "kind": "embedding", "rows": 611, "table": 87, "dim": 64, "scale": 1.0,
         "padded": 0.0, "dtype": "float32"},
        # element-pair rows of a large batch's edges, padded edges among them
        {"name": "embedding_edges", "kind": "embedding", "rows": 400000, "table": 7569, "dim": 128, "scale": 0.5,
         "padded": 0.02, "dtype": "float32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = {}
    for c in listed():
        w = work(c)
        top[c["kind"]] = {k: max(w[k], top.get(c["kind"], w)[k]) for k in w}
    while True:
        kind = rng.choice(ATTENTION + ("attention_train", "dropout", "embedding"))
        dtype = "float64" if rng.random() < 0.2 else "float32"
        if kind == "dropout":
            shared = 1 if rng.random() < 0.4 else rng.choice([4, 9, 16, 25, 49])
            c = {"kind": kind, "rows": _log(rng, 1, 500000), "shared": shared, "inner": _log(rng, 1, 512),
                 "p": rng.choice([0.05, 0.1, 0.2, 0.5]), "dtype": dtype}
        elif kind == "embedding":
            c = {"kind": kind, "rows": _log(rng, 1, 400000), "table": _log(rng, 5, 8000), "dim": _log(rng, 1, 512),
                 "scale": rng.choice([1.0, 0.5]), "padded": rng.choice([0.0, 0.02]), "dtype": dtype}
        else:
            lo = _log(rng, 4, 2000)
            hi = min(8000, int(lo * rng.uniform(1.0, 4.0)))
            kv = rng.choice([1, 1, 2, 4])
            c = {"kind": kind, "structures": _log(rng, 1, 512), "lo": lo, "hi": hi, "heads": kv * rng.choice([1, 1, 2, 4]),
                 "kv_heads": kv, "dim": rng.choice([8, 16, 20, 24, 32, 48, 50, 64, 96, 128]), "dtype": dtype,
                 "masked": rng.choice([0.0, 0.0, 0.1]) if lo >= 8 else 0.0, "tail": rng.choice([0, 0, 5])}
            padded = c["structures"] * hi * hi * c["heads"]
            if padded > 6e8 or (dtype == "float64" and padded > 1e8):
                continue
        if all(v <= top[kind][k] for k, v in work(c).items()):
            return c


@functools.lru_cache(maxsize=64)
def _sizes(structures, lo, hi):
    rng = random.Random(1000003 * structures + 1009 * lo + hi)
    return [rng.randint(lo, hi) for _ in range(structures)]


def _lengths(case):
    return _sizes(case["structures"], case["lo"], case["hi"])


def work(case):
    w = 8 if case["dtype"] == "float64" else 4
    kind = case["kind"]
    if kind == "dropout":
        n = case["rows"] * case["shared"] * case["inner"]
        return {"bytes": 4 * n * w, "flops": 2 * n}  # x and y, the gradient in and out
    if kind == "embedding":
        n, c = case["rows"], case["dim"]
        return {"bytes": 2 * n * c * w + 2 * case["table"] * c * w + 2 * n * 8, "flops": 2 * n * c}
    lens = _lengths(case)
    n, pairs = sum(lens) + case["tail"], sum(x * x for x in lens)
    rows_q, rows_k = n * case["heads"] * case["dim"], n * case["kv_heads"] * case["dim"]
    # q, o and k, v; with do and dq, dk, dv; with the three cotangents and the four second gradients
    q_rows, k_rows, products = {"attention": (2, 2, 2), "attention_train": (4, 4, 7),
                                "attention_force_train": (7, 8, 19)}[kind]
    return {"bytes": w * (q_rows * rows_q + k_rows * rows_k),
            "flops": 2 * products * pairs * case["heads"] * case["dim"]}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def prepare(case, seed):
    g = _generator(seed)
    dt = DTYPES[case["dtype"]]
    kind = case["kind"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt)

    if kind == "dropout":
        shape = (case["rows"], case["shared"], case["inner"])
        rng = torch.randint(0, 2 ** 62, (2,), generator=g, device="cuda", dtype=torch.int64)
        return {"case": case, "x": normal(*shape), "gy": normal(*shape), "rng": rng}
    if kind == "embedding":
        # a few elements are most of the atoms: the id's logarithm is uniform
        u = torch.rand(case["rows"], generator=g, device="cuda", dtype=torch.float64)
        ids = (torch.exp(u * math.log(case["table"] + 1.0)) - 1.0).long().clamp(0, case["table"] - 1)
        if case["padded"]:
            off = torch.rand(case["rows"], generator=g, device="cuda") < case["padded"]
            ids = torch.where(off, torch.full_like(ids, -1), ids)
        return {"case": case, "table": normal(case["table"], case["dim"]), "ids": ids,
                "gy": normal(case["rows"], case["dim"])}
    lens = _lengths(case)
    n, h, hk, d = sum(lens) + case["tail"], case["heads"], case["kv_heads"], case["dim"]
    s = {"case": case, "q": normal(n, h, d), "k": normal(n, hk, d), "v": normal(n, hk, d), "max_len": max(lens),
         "ptr": torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int64, device="cuda"), "mask": None}
    if case["masked"]:
        s["mask"] = torch.rand(n, generator=g, device="cuda") >= case["masked"]
    if kind != "attention":
        s["do"] = normal(n, h, d)
    if kind == "attention_force_train":
        s["cq"], s["ck"], s["cv"] = normal(n, h, d), normal(n, hk, d), normal(n, hk, d)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _padded(state):
    """The row of each padded slot (B, L), which slots hold an atom, and each atom's slot."""
    ptr, most, n = state["ptr"], state["max_len"], state["q"].shape[0]
    row = ptr[:-1, None] + torch.arange(most, device=ptr.device)
    return row.clamp(max=n - 1), row < ptr[1:, None], row


def _pad(t, row, on, groups):
    """(N, Hk, D) to (B, Hk * groups, L, D), zero in the empty slots; in 32 bits at least."""
    x = torch.where(on[..., None, None], t[row], 0.0).transpose(1, 2)
    return x if groups == 1 else x.repeat_interleave(groups, 1)


def _unpad(x, state, row, on, heads):
    """(B, H, L, D) back to (N, heads, D), summed over the heads that share; rows of no structure are zero."""
    if x.shape[1] != heads:
        x = x.view(x.shape[0], heads, -1, x.shape[2], x.shape[3]).sum(2)
    out = x.new_zeros(state["q"].shape[0], heads, x.shape[3])
    out[row[on]] = x.transpose(1, 2)[on]
    return out


def _probabilities(q, k, scale, keys):
    """Row softmax over the allowed keys; zero rows where there are none."""
    s = torch.where(keys, (q * scale) @ k.transpose(2, 3), -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0)


def _plain_attention(state):
    case = state["case"]
    h, hk = case["heads"], case["kv_heads"]
    groups, scale = h // hk, case["dim"] ** -0.5
    row, on, whole = _padded(state)
    keys = on if state["mask"] is None else on & state["mask"][row]
    keys = keys[:, None, None, :]
    q, k, v = _pad(state["q"], row, on, 1), _pad(state["k"], row, on, groups), _pad(state["v"], row, on, groups)
    p = _probabilities(q, k, scale, keys)
    o = p @ v
    out = {"o": _unpad(o, state, whole, on, h)}
    if case["kind"] == "attention":
        return out
    do = _pad(state["do"], row, on, 1)
    dp = do @ v.transpose(2, 3)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    out["dq"] = _unpad(scale * (ds @ k), state, whole, on, h)
    out["dk"] = _unpad(scale * (ds.transpose(2, 3) @ q), state, whole, on, hk)
    out["dv"] = _unpad(p.transpose(2, 3) @ do, state, whole, on, hk)
    if case["kind"] == "attention_train":
        return out
    a, b, c = _pad(state["cq"], row, on, 1), _pad(state["ck"], row, on, groups), _pad(state["cv"], row, on, groups)
    t = scale * (a @ k.transpose(2, 3) + q @ b.transpose(2, 3))
    r = (p * t).sum(-1, keepdim=True)
    e = t * dp + do @ c.transpose(2, 3) - t * delta - r * dp
    m = p * (e - (p * e).sum(-1, keepdim=True))
    pt = p * (t - r)
    out["q2"] = _unpad(scale * (m @ k + ds @ b), state, whole, on, h)
    out["k2"] = _unpad(scale * (m.transpose(2, 3) @ q + ds.transpose(2, 3) @ a), state, whole, on, hk)
    out["v2"] = _unpad(pt.transpose(2, 3) @ do, state, whole, on, hk)
    out["do2"] = _unpad(pt @ v + p @ c, state, whole, on, h)
    return out


def _product(m, x):
    """High and low 32 bits of m * x for a constant m and x (int64), both below 2^32."""
    t = m * (x & 0xFFFF)
    u = m * (x >> 16) + (t >> 16)
    return u >> 16, ((u & 0xFFFF) << 16) | (t & 0xFFFF)


def _philox_round(s, _):
    c0, c1, c2, c3, k0, k1 = s
    h0, l0 = _product(0xD2511F53, c0)
    h1, l1 = _product(0xCD9E8D57, c2)
    return h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0, (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF


def _plain_dropout(state):
    case, x = state["case"], state["x"]
    n = case["rows"] * case["inner"]
    seed, offset = state["rng"][0], state["rng"][1]
    i = torch.arange((n + 3) // 4, device=x.device, dtype=torch.int64)
    start = (i & 0xFFFFFFFF, i >> 32, (offset & 0xFFFFFFFF).expand_as(i), ((offset >> 32) & 0xFFFFFFFF).expand_as(i),
             seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF)
    words = functools.reduce(_philox_round, range(10), start)[:4]
    bits = torch.stack(words, 1).view(-1)[:n].view(case["rows"], 1, case["inner"])
    keep = bits >= int(case["p"] * 2 ** 32)
    factor = 1.0 / (1.0 - case["p"])
    return {"y": torch.where(keep, x * factor, 0.0), "dx": torch.where(keep, state["gy"] * factor, 0.0)}


def _plain_embedding(state):
    case, table, ids = state["case"], state["table"], state["ids"]
    on = ids >= 0
    at = ids.clamp(min=0)
    out = torch.where(on[:, None], case["scale"] * table[at], 0.0)
    g = torch.where(on[:, None], state["gy"], 0.0).double()
    grad = case["scale"] * torch.zeros(table.shape, dtype=torch.float64, device=table.device).index_add(0, at, g)
    return {"out": out, "dtable": grad.to(table.dtype)}


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return {"dropout": _plain_dropout, "embedding": _plain_embedding}.get(kind, _plain_attention)(state)
    from xnn_b200.ops import counter_dropout, embedding_lookup, structure_attention
    if kind == "dropout":
        x = state["x"].detach().requires_grad_()
        y = counter_dropout(x, case["p"], state["rng"], shared=(1,))
        return {"y": y, "dx": torch.autograd.grad(y, x, state["gy"])[0]}
    if kind == "embedding":
        table = state["table"].detach().requires_grad_()
        out = embedding_lookup(table, state["ids"], scale=case["scale"])
        return {"out": out, "dtable": torch.autograd.grad(out, table, state["gy"])[0]}
    q, k, v = state["q"], state["k"], state["v"]
    if kind == "attention":
        return {"o": structure_attention(q, k, v, state["ptr"], max_len=state["max_len"], key_mask=state["mask"])}
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = structure_attention(q, k, v, state["ptr"], max_len=state["max_len"], key_mask=state["mask"])
    if kind == "attention_train":
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), state["do"])
        return {"o": o, "dq": dq, "dk": dk, "dv": dv}
    do = state["do"].detach().requires_grad_()
    first = torch.autograd.grad(o, (q, k, v), do, create_graph=True)
    second = torch.autograd.grad(first, (q, k, v, do), (state["cq"], state["ck"], state["cv"]))
    return dict(zip(("o", "dq", "dk", "dv", "q2", "k2", "v2", "do2"), (o,) + first + second))


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_structure(q, k, v, keys, scale):
    """One structure, heads first: softmax over the allowed keys by its definition."""
    s = torch.einsum("ihd,jhd->hij", q, k) * scale
    return torch.einsum("hij,jhd->ihd", torch.softmax(s[:, :, keys], -1), v[keys])


def _exact_attention(state):
    case = state["case"]
    h, hk, kind = case["heads"], case["kv_heads"], case["kind"]
    scale, n = case["dim"] ** -0.5, state["q"].shape[0]
    rows = {}
    at = 0
    for length in _lengths(case):
        part = slice(at, at + length)
        at += length

        def take(name):
            return state[name][part].double().detach().requires_grad_()
        q, k, v = take("q"), take("k"), take("v")
        keys = (torch.ones(length, dtype=torch.bool, device=q.device) if state["mask"] is None else state["mask"][part])
        got = {"o": torch.zeros_like(q)}
        if bool(keys.any()):
            wide = torch.arange(h, device=q.device) // (h // hk)
            o = _exact_structure(q, k[:, wide], v[:, wide], keys, scale)
            got = {"o": o}
            if kind != "attention":
                do = take("do")
                more = kind == "attention_force_train"
                first = torch.autograd.grad(o, (q, k, v), do, create_graph=more)
                got.update(zip(("dq", "dk", "dv"), first))
                if more:
                    second = torch.autograd.grad(first, (q, k, v, do), (take("cq"), take("ck"), take("cv")))
                    got.update(zip(("q2", "k2", "v2", "do2"), second))
        for name, value in got.items():
            heads = hk if name in ("dk", "dv", "k2", "v2") else h
            if name not in rows:
                rows[name] = torch.zeros(n, heads, case["dim"], dtype=torch.float64, device=q.device)
            rows[name][part] = value.detach()
    return rows


def _exact_dropout(state):
    case = state["case"]
    n = case["rows"] * case["inner"]
    if n > 8_000_000:
        return None
    low = np.uint64(0xFFFFFFFF)
    seed, offset = (int(v) for v in state["rng"].cpu())
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    c = [block & low, block >> np.uint64(32), np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(key[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    keep = np.stack(c, 1).reshape(-1)[:n] >= np.uint64(int(case["p"] * 2 ** 32))
    mask = torch.from_numpy(keep).to(state["x"].device).view(case["rows"], 1, case["inner"])
    return {"y": mask * state["x"].double() / (1.0 - case["p"]), "dx": mask * state["gy"].double() / (1.0 - case["p"])}


def _exact_embedding(state):
    case, ids = state["case"], state["ids"].cpu().numpy()
    table, gy = state["table"].double(), state["gy"].double()
    # one row of zeros behind the table for the padded ids; the gradient as differences of a running sum is too
    # coarse for long runs, so each id's rows are summed from the sorted order
    longer = torch.cat([table, torch.zeros_like(table[:1])])
    where = torch.from_numpy(np.where(ids < 0, case["table"], ids)).to(table.device)
    order = torch.argsort(where, stable=True)
    counts = torch.bincount(where, minlength=case["table"] + 1).cpu().tolist()
    grad = torch.stack([part.sum(0) for part in torch.split(gy[order], counts)])[:case["table"]]
    return {"out": case["scale"] * longer[where], "dtable": case["scale"] * grad}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "dropout":
        return _exact_dropout(state)
    if case["kind"] == "embedding":
        return _exact_embedding(state)
    return _exact_attention(state)
