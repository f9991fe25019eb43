"""Workloads of the expert-routing operators: sort + dispatch, combine (and gradient), the experts' products with their
epilogue, and the products' gradients.

A case is a dict of plain values; ``prepare`` makes its inputs on the GPU from a seed, ``run`` makes one pass, in the
operators' plain form (elementary torch operations in 32 bits, rounded once at the end) or, with ``own`` set, through
library_b200.api.  ``exact`` computes the same outputs in 64 bits, written apart from the plain form.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---- cases -----------------------------------------------------------------------------------

def listed():
    return [
        # a serving step of four sequences, two experts each
        dict(name="sort_decode", kind="sort", tokens=4, topk=2, experts=8, width=1024, dtype="bf16", dropped=0.0, ids="i64"),
        # a prefill batch, fine-grained experts
        dict(name="sort_prefill", kind="sort", tokens=8192, topk=8, experts=64, width=2048, dtype="bf16", dropped=0.0, ids="i32"),
        # a padded fp32 batch (padding tokens route nowhere), odd sizes throughout
        dict(name="sort_padded_odd", kind="sort", tokens=3001, topk=3, experts=61, width=1003, dtype="fp32", dropped=0.15, ids="i64"),
        # back to token order with the gate weights, added to the residual stream: one serving step
        dict(name="combine_decode", kind="combine", tokens=7, topk=4, experts=16, width=4096, dtype="bf16", dropped=0.0, residual=True),
        # the same for a prefill batch
        dict(name="combine_prefill", kind="combine", tokens=8192, topk=8, experts=64, width=2048, dtype="bf16", dropped=0.05, residual=True),
        # its gradient in a training step: dYs and the gate weights' gradient
        dict(name="combine_grad_train", kind="combine_grad", tokens=8192, topk=6, experts=64, width=2048, dtype="bf16", dropped=0.0),
        # one token through its eight experts: the weights' bytes
        dict(name="product_token", kind="product", rows=8, experts=64, k=2048, n=1408, dtype="bf16", op="T", act="silu", bias=True,
             residual=False, preact=False, tail=0),
        # a dense layer (one segment) for a small decode batch with the residual in the epilogue
        dict(name="product_dense_decode", kind="product", rows=17, experts=1, k=4096, n=4096, dtype="fp16", op="T", act="none", bias=True,
             residual=True, preact=False, tail=0),
        # a training step's up projection over ragged segments: saves Z for the backward pass
        dict(name="product_train", kind="product", rows=32768, experts=32, k=2048, n=4096, dtype="bf16", op="T", act="gelu", bias=True,
             residual=False, preact=True, tail=300),
        # the activation's gradient and the bias gradient
        dict(name="act_grad_train", kind="act_grad", rows=32768, experts=32, n=4096, dtype="bf16", act="silu"),
        # the products' gradients, a training step
        dict(name="product_grad_train", kind="product_grad", rows=32768, experts=16, k=2048, n=2048, dtype="bf16", op="T"),
        # the same over few ragged rows, odd sizes, weights stored K x N
        dict(name="product_grad_ragged_odd", kind="product_grad", rows=1777, experts=7, k=1000, n=515, dtype="fp16", op="N"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A width: mostly a multiple of 8, now and then any number."""
    v = _log_int(rng, lo, hi)
    return v if rng.random() < 0.3 else max(8, v // 8 * 8)


def draw(rng):
    kind = rng.choice(["sort", "combine", "combine_grad", "product", "product", "act_grad", "product_grad"])
    if kind in ("sort", "combine", "combine_grad"):
        most = 8192 * 8 * 2048 * 2 if kind == "sort" else 8192 * 6 * 2048 * 2
        while True:
            c = dict(kind=kind, tokens=_log_int(rng, 1, 16384), topk=rng.randint(1, 8), experts=_log_int(rng, 8, 256),
                     width=_size(rng, 64, 4096), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                     dropped=rng.choice([0.0, 0.0, 0.1, 0.5]))
            if c["tokens"] * c["topk"] * c["width"] * SIZE[c["dtype"]] <= most:
                break
        if kind == "sort":
            c["ids"] = rng.choice(["i32", "i64"])
        if kind == "combine":
            c["residual"] = rng.random() < 0.5
        return c
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    while True:
        rows, experts, n = _log_int(rng, 1, 32768), _log_int(rng, 1, 64), _size(rng, 64, 4096)
        if kind == "act_grad":
            return dict(kind=kind, rows=rows, experts=experts, n=n, dtype=dtype, act=rng.choice(["none", "relu", "gelu", "silu"]))
        k = _size(rng, 64, 4096)
        most = 32768 * 2048 * (4096 if kind == "product" else 2048)
        if rows * k * n <= most and experts * k * n <= 32 * 2048 * 4096:
            break
    c = dict(kind=kind, rows=rows, experts=experts, k=k, n=n, dtype=dtype, op=rng.choice(["T", "T", "N"]))
    if kind == "product":
        c.update(act=rng.choice(["none", "relu", "gelu", "silu"]), bias=rng.random() < 0.7, residual=rng.random() < 0.4,
                 preact=rng.random() < 0.3, tail=rng.choice([0, 0, rng.randint(1, 200)]) if rows > max(experts, 200) else 0)
    return c


# ---- inputs ----------------------------------------------------------------------------------

def _route(case, g):
    """Expert ids (tokens x topk) with uneven popularity, distinct within a token; dropped tokens route nowhere (-1)."""
    t, k, e = case["tokens"], case["topk"], case["experts"]
    popular = torch.randn(e, device="cuda", generator=g) * 0.7
    gumbel = -torch.log(-torch.log(torch.rand(t, e, device="cuda", generator=g).clamp(1e-9, 1 - 1e-7)))
    ids = torch.topk(gumbel + popular, k, dim=1).indices
    if case["dropped"]:
        ids = torch.where((torch.rand(t, 1, device="cuda", generator=g) < case["dropped"]), torch.full_like(ids, -1), ids)
    return ids


def _positions(ids, experts):
    """The stable sort by expert: offsets (experts + 1) and every slot's sorted position (-1: dropped)."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    order = torch.sort(key, stable=True).indices
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=order.device)
    position = torch.where(key < experts, position, torch.full_like(position, -1))
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device)
    offsets[1:] = torch.cumsum((key[:, None] == torch.arange(experts, device=ids.device)[None, :]).sum(0), 0)
    return offsets.int(), position.int().reshape(ids.shape)


def _segments(case, g):
    """Rows per expert, as offsets: distinct experts for no more rows than experts (one token's choice), else a draw
    with uneven popularity in which an expert may stay empty."""
    rows, e = case["rows"], case["experts"]
    tail = case.get("tail", 0)
    if rows <= e:
        pick = torch.randperm(e, device="cuda", generator=g)[:rows]
    else:
        p = torch.softmax(torch.randn(e, device="cuda", generator=g) * 0.5, 0)
        pick = torch.multinomial(p, max(rows - tail, 1), replacement=True, generator=g)
    off = torch.zeros(e + 1, dtype=torch.int64, device="cuda")
    off[1:] = torch.cumsum(torch.bincount(pick, minlength=e), 0)
    return off.int()


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    s = dict(case=case)
    kind = case["kind"]
    if kind in ("sort", "combine", "combine_grad"):
        t, k, e, h = case["tokens"], case["topk"], case["experts"], case["width"]
        ids = _route(case, g)
        if kind == "sort":
            s["ids"] = ids.int() if case["ids"] == "i32" else ids
            s["x"] = normal(t, h)
            return s
        s["ids"] = ids.int()
        s["offsets"], s["position"] = _positions(ids, e)
        s["ys"] = normal(t * k, h)
        s["w"] = torch.softmax(torch.randn(t, k, device="cuda", generator=g), 1)
        if kind == "combine":
            s["r"] = normal(t, h) if case["residual"] else None
        else:
            s["dy"] = normal(t, h, scale=0.1)
        return s
    off = _segments(case, g)
    s["offsets"], s["counts"] = off, [int(v) for v in (off[1:] - off[:-1]).tolist()]
    rows, e, n = case["rows"], case["experts"], case["n"]
    if kind == "act_grad":
        s["dy"] = normal(rows, n, scale=0.1)
        s["z"] = normal(rows, n, scale=1.5) if case["act"] != "none" else None
        return s
    k = case["k"]
    s["x"] = normal(rows, k)
    s["w"] = normal(e * n, k, scale=k ** -0.5) if case["op"] == "T" else normal(e * k, n, scale=k ** -0.5)
    if kind == "product":
        s["b"] = normal(e, n, scale=0.3) if case["bias"] else None
        s["r"] = normal(rows, n) if case["residual"] else None
    else:
        s["dz"] = normal(rows, n, scale=0.1)
    return s


def prepare(case, seed):
    """The inputs, and what a program keeps beside them: output buffers (rows behind the last segment stay as they are,
    here zero) and, for the library's calls, the handle, the descriptors and the workspaces."""
    s = _inputs(case, seed)
    dt = DTYPES[case["dtype"]]
    kind = case["kind"]

    def zeros(*shape, dtype=dt):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    if kind == "sort":
        s["out"] = [zeros(case["tokens"] * case["topk"], case["width"])]
    elif kind == "combine":
        s["out"] = [zeros(case["tokens"], case["width"])]
    elif kind == "combine_grad":
        s["out"] = [zeros(case["tokens"] * case["topk"], case["width"]), zeros(case["tokens"], case["topk"], dtype=torch.float32)]
    elif kind == "product":
        s["out"] = [zeros(case["rows"], case["n"])] + ([zeros(case["rows"], case["n"])] if case["preact"] else [])
    elif kind == "act_grad":
        s["out"] = [zeros(case["rows"], case["n"]), zeros(case["experts"], case["n"], dtype=torch.float32)]
    else:
        s["out"] = [zeros(case["rows"], case["k"]), zeros(*s["w"].shape)]
    if own:
        _describe(s)
    return s


def _describe(s):
    from library_b200 import api
    case, out, kind = s["case"], s["out"], s["case"]["kind"]
    h = s["handle"] = api.Handle()
    d = s["d"] = {}

    def workspace(size):
        return torch.empty(size, dtype=torch.uint8, device="cuda") if size else None

    for name in ("x", "ys", "r", "dy", "w", "b", "z", "dz"):
        if s.get(name) is not None and not (name == "w" and kind.startswith("combine")):
            d[name] = api.DnMat(s[name])
    d["out"] = [api.DnMat(t) for t in out if not (kind == "combine_grad" and t is out[1])]
    if kind == "sort":
        s["routing"] = api.Routing(s["ids"], case["experts"])
        s["buffer"] = workspace(api.routing_buffer_size(h, s["routing"]))
    elif kind in ("combine", "combine_grad"):
        s["routing"] = api.Routing(s["ids"], case["experts"], s["offsets"], s["position"])
    else:
        # one segment over all rows is a plain dense layer: no offsets needed
        s["seg"] = None if case["experts"] == 1 and sum(s["counts"]) == case["rows"] else s["offsets"]
        act = s["act"] = {"none": api.ACT_NONE, "relu": api.ACT_RELU, "gelu": api.ACT_GELU, "silu": api.ACT_SILU}[case.get("act", "none")]
        if kind == "product":
            s["op"] = api.OP_T if case["op"] == "T" else api.OP_N
            s["buffer"] = workspace(api.expert_mm_buffer_size(h, d["x"], d["w"], d["out"][0], s["seg"], s["op"]))
        elif kind == "act_grad":
            s["buffer"] = workspace(api.expert_act_grad_buffer_size(h, d["dy"], s["seg"], act, d["out"][1]))
        else:
            s["op"], s["back"] = (api.OP_T, api.OP_N) if case["op"] == "T" else (api.OP_N, api.OP_T)
            s["buffer"] = workspace(max(api.expert_mm_buffer_size(h, d["dz"], d["w"], d["out"][0], s["seg"], s["back"]),
                                        api.expert_mm_grad_weight_buffer_size(h, d["x"], d["dz"], d["out"][1], s["seg"], s["op"])))


# ---- one pass --------------------------------------------------------------------------------

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from library_b200 import api
    h, d, out, kind = s["handle"], s["d"], s["out"], s["case"]["kind"]
    h.use_torch_stream()
    if kind == "sort":
        r = s["routing"]
        api.routing_sort(h, r, s["buffer"])
        api.routing_dispatch(h, r, d["x"], d["out"][0])
        return [r.offsets, r.position, out[0]]
    if kind == "combine":
        api.routing_combine(h, s["routing"], d["ys"], d["out"][0], s["w"], d.get("r"))
        return out
    if kind == "combine_grad":
        api.routing_combine_grad(h, s["routing"], d["dy"], d["ys"], d["out"][0], s["w"], out[1])
        return out
    if kind == "product":
        api.expert_mm(h, d["x"], d["w"], d["out"][0], s["seg"], s["op"], d.get("b"), s["act"], d.get("r"),
                      d["out"][1] if len(out) > 1 else None, s["buffer"])
        return out
    if kind == "act_grad":
        api.expert_act_grad(h, d["dy"], d.get("z"), d["out"][0], s["seg"], s["act"], d["out"][1], s["buffer"])
        return out
    api.expert_mm(h, d["dz"], d["w"], d["out"][0], s["seg"], s["back"], buffer=s["buffer"])
    api.expert_mm_grad_weight(h, d["x"], d["dz"], d["out"][1], s["seg"], s["op"], s["buffer"])
    return out


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * torch.erfc(z * -(0.5 ** 0.5))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * torch.erfc(z * -(0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    p = 1 / (1 + torch.exp(-z))
    return p * (1 + z * (1 - p))


def _run_plain(s):
    case, out, kind = s["case"], s["out"], s["case"]["kind"]
    dt = DTYPES[case["dtype"]]
    if kind == "sort":
        offsets, position = _positions(s["ids"], case["experts"])
        flat = position.reshape(-1).long()
        t = torch.arange(case["tokens"], device="cuda").repeat_interleave(case["topk"])
        xs = torch.zeros_like(out[0])
        # dropped slots write to a row of their own behind the sorted ones, which is not returned
        xs = torch.cat([xs, xs.new_zeros(1, case["width"])])
        xs[torch.where(flat >= 0, flat, torch.full_like(flat, flat.numel()))] = s["x"][t]
        return [offsets, position, xs[:-1]]
    if kind == "combine":
        y = s["r"].float() if s["r"] is not None else torch.zeros(out[0].shape, device="cuda")
        for j in range(case["topk"]):
            p = s["position"][:, j].long()
            row = s["ys"][p.clamp(min=0)].float() * s["w"][:, j:j + 1]
            y = y + torch.where((p >= 0)[:, None], row, torch.zeros_like(row))
        return [y.to(dt)]
    if kind == "combine_grad":
        dys = torch.zeros(case["tokens"] * case["topk"] + 1, case["width"], dtype=dt, device="cuda")
        dw = torch.zeros_like(out[1])
        dy = s["dy"].float()
        for j in range(case["topk"]):
            p = s["position"][:, j].long()
            dot = (dy * s["ys"][p.clamp(min=0)].float()).sum(1)
            dw[:, j] = torch.where(p >= 0, dot, torch.zeros_like(dot))
            dys[torch.where(p >= 0, p, torch.full_like(p, dys.shape[0] - 1))] = (dy * s["w"][:, j:j + 1]).to(dt)
        return [dys[:-1], dw]
    outs = [torch.zeros_like(t) for t in out]
    lo = 0
    for e, count in enumerate(s["counts"]):
        hi = lo + count
        if kind == "act_grad":
            dz = s["dy"][lo:hi].float()
            if s["z"] is not None:
                dz = dz * _act_slope(s["z"][lo:hi].float(), case["act"])
            outs[0][lo:hi] = dz.to(dt)
            outs[1][e] = dz.sum(0)
        elif kind == "product" and count:
            size = case["n"] if case["op"] == "T" else case["k"]
            w = s["w"][e * size:(e + 1) * size].float()
            z = torch.matmul(s["x"][lo:hi].float(), w.t() if case["op"] == "T" else w)
            if s["b"] is not None:
                z = z + s["b"][e].float()
            if case["preact"]:
                outs[1][lo:hi] = z.to(dt)
            y = _act(z, case["act"])
            if s["r"] is not None:
                y = y + s["r"][lo:hi].float()
            outs[0][lo:hi] = y.to(dt)
        elif kind == "product_grad" and count:
            size = case["n"] if case["op"] == "T" else case["k"]
            w, dz, x = s["w"][e * size:(e + 1) * size].float(), s["dz"][lo:hi].float(), s["x"][lo:hi].float()
            if case["op"] == "T":
                outs[0][lo:hi] = torch.matmul(dz, w).to(dt)
                outs[1][e * size:(e + 1) * size] = torch.matmul(dz.t(), x).to(dt)
            else:
                outs[0][lo:hi] = torch.matmul(dz, w.t()).to(dt)
                outs[1][e * size:(e + 1) * size] = torch.matmul(x.t(), dz).to(dt)
        lo = hi
    return outs


# ---- what a pass cannot do without ------------------------------------------------------------

def work(case):
    z = SIZE[case["dtype"]]
    if case["kind"] in ("sort", "combine", "combine_grad"):
        t, slots, h = case["tokens"], case["tokens"] * case["topk"], case["width"]
        kept = slots * (1 - case["dropped"])
        if case["kind"] == "sort":
            return {"bytes": int(slots * ((4 if case["ids"] == "i32" else 8) + 4) + 4 * (case["experts"] + 1) + t * h * z + kept * h * z),
                    "flops": 0}
        if case["kind"] == "combine":
            return {"bytes": int(slots * 8 + kept * h * z + t * h * z * (2 if case["residual"] else 1)), "flops": int(2 * kept * h)}
        return {"bytes": int(slots * 12 + t * h * z + 2 * kept * h * z), "flops": int(3 * kept * h)}
    rows, e, n = max(case["rows"] - case.get("tail", 0), 1), case["experts"], case["n"]
    if case["kind"] == "act_grad":
        return {"bytes": int(rows * n * z * (2 if case["act"] == "none" else 3) + e * n * 4), "flops": int(rows * n * 2)}
    k = case["k"]
    touched = rows if rows <= e else e * (1 - (1 - 1 / e) ** rows)  # weights read: of the experts with rows
    if case["kind"] == "product":
        return {"bytes": int(rows * k * z + touched * n * k * z + touched * n * z * case["bias"]
                             + rows * n * z * (1 + case["residual"] + case["preact"])), "flops": int(2 * rows * n * k)}
    # inputs X, dZ and the touched weights once; dX and every expert's dW written
    return {"bytes": int(rows * (2 * k + n) * z + touched * n * k * z + e * n * k * z), "flops": int(4 * rows * n * k)}


# ---- the definition in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    kind, dev = case["kind"], "cuda"
    if kind in ("sort", "combine", "combine_grad"):
        t, k, h = case["tokens"], case["topk"], case["width"]
        ids = s["ids"].cpu().long().numpy().reshape(-1)
        # slot by slot, as the definition says: first the experts' sizes, then places in slot order
        counts = [0] * case["experts"]
        for i in ids:
            if 0 <= i < case["experts"]:
                counts[i] += 1
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        nxt, place = list(starts), [-1] * len(ids)
        for slot, i in enumerate(ids):
            if 0 <= i < case["experts"]:
                place[slot] = nxt[i]
                nxt[i] += 1
        position = torch.tensor(place, dtype=torch.int32, device=dev).reshape(t, k)
        kept = position >= 0
        token, choice = torch.nonzero(kept, as_tuple=True)
        rows = position[kept].long()
        if kind == "sort":
            xs = torch.zeros(t * k, h, dtype=torch.float64, device=dev)
            xs.index_copy_(0, rows, s["x"].double().index_select(0, token))
            return [torch.tensor(starts, dtype=torch.int32, device=dev), position, xs]
        w = s["w"].double()[token, choice][:, None]
        if kind == "combine":
            y = torch.zeros(t, h, dtype=torch.float64, device=dev)
            y.index_add_(0, token, s["ys"].double().index_select(0, rows) * w)
            return [y if s["r"] is None else y + s["r"].double()]
        dys = torch.zeros(t * k, h, dtype=torch.float64, device=dev)
        dyt = s["dy"].double().index_select(0, token)
        dys.index_copy_(0, rows, dyt * w)
        dw = torch.zeros(t, k, dtype=torch.float64, device=dev)
        dw[token, choice] = torch.einsum("rh,rh->r", dyt, s["ys"].double().index_select(0, rows))
        return [dys, dw]
    off = s["offsets"].tolist()
    rows, n, e = case["rows"], case["n"], case["experts"]

    def normal_cdf(v):
        return torch.special.ndtr(v)

    if kind == "act_grad":
        dz = s["dy"].double()
        if s["z"] is not None:
            z = s["z"].double()
            dz = dz * {"relu": lambda: (z > 0).double(),
                       "gelu": lambda: normal_cdf(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi),
                       "silu": lambda: torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)}[case["act"]]()
        dz[off[-1]:] = 0
        db = torch.stack([dz[a:b].sum(0) for a, b in zip(off, off[1:])])
        return [dz, db]
    k = case["k"]
    w3 = s["w"].double().reshape(e, n, k) if case["op"] == "T" else s["w"].double().reshape(e, k, n).transpose(1, 2)
    if kind == "product":
        z = torch.zeros(rows, n, dtype=torch.float64, device=dev)
        for i, (a, b) in enumerate(zip(off, off[1:])):
            z[a:b] = torch.einsum("rk,nk->rn", s["x"][a:b].double(), w3[i])
            if s["b"] is not None:
                z[a:b] += s["b"][i].double()
        y = {"none": lambda: z.clone(), "relu": lambda: z.clamp(min=0), "gelu": lambda: z * normal_cdf(z),
             "silu": lambda: z * torch.sigmoid(z)}[case["act"]]()
        if s["r"] is not None:
            y = y + s["r"].double()
        y[off[-1]:] = 0
        return [y, z] if case["preact"] else [y]
    dx = torch.zeros(rows, k, dtype=torch.float64, device=dev)
    dw = torch.zeros(e, n, k, dtype=torch.float64, device=dev)
    for i, (a, b) in enumerate(zip(off, off[1:])):
        dx[a:b] = torch.einsum("rn,nk->rk", s["dz"][a:b].double(), w3[i])
        dw[i] = torch.einsum("rn,rk->nk", s["dz"][a:b].double(), s["x"][a:b].double())
    return [dx, dw.reshape(e * n, k) if case["op"] == "T" else dw.transpose(1, 2).reshape(e * k, n).contiguous()]
