"""The operators at the two ends of a language model's training step, in their plain form and as calls of the
library: embedding lookup and its gradient, dropout from a counter-based generator, and the cross entropy of a linear
output layer with its gradients.

Each case names an operator ("op") and its sizes; `run` makes one pass of it."""
import ctypes
import math

import torch

own = False

TYPES = {"float32": (torch.float32, 0), "float16": (torch.float16, 2), "bfloat16": (torch.bfloat16, 4)}
IGNORE = -100


# ------------------------------------------------------------------------------------------------ the cases ----
def listed():
    return [
        # one generated token enters the model: latency
        {"name": "lookup, one token", "op": "lookup", "tokens": 1, "vocab": 32000, "dim": 4096, "type": "float16", "p": 0.0},
        # a training batch enters the model, with embedding dropout
        {"name": "lookup, batch, dropout", "op": "lookup", "tokens": 8192, "vocab": 131072, "dim": 4096, "type": "bfloat16", "p": 0.1},
        # mixed precision: fp16 in, fp16 gradient of the table for the mixed-precision step
        {"name": "table gradient, half", "op": "table_gradient", "tokens": 8192, "vocab": 32000, "dim": 4096, "type": "float16",
         "out": "float16", "p": 0.0, "add": False},
        # tied weights: the table's gradient is added to what the output layer left there; odd sizes
        {"name": "table gradient, tied, odd", "op": "table_gradient", "tokens": 4097, "vocab": 50001, "dim": 1000, "type": "float32",
         "out": "float32", "p": 0.0, "add": True},
        # the largest batch, with the embedding's dropout, into an fp32 gradient for the fp32 steps
        {"name": "table gradient, large", "op": "table_gradient", "tokens": 32768, "vocab": 131072, "dim": 2048, "type": "bfloat16",
         "out": "float32", "p": 0.1, "add": False},
        # a small fp32 activation
        {"name": "dropout, small", "op": "dropout", "elements": 257000, "type": "float32", "p": 0.5, "residual": False},
        # the end of a transformer block: residual + dropout(x)
        {"name": "dropout, residual", "op": "dropout", "elements": 8192 * 4096, "type": "float16", "p": 0.1, "residual": True},
        # its backward pass (the same call on the gradient), an odd number of elements
        {"name": "dropout, backward, odd", "op": "dropout", "elements": 16383 * 4099, "type": "bfloat16", "p": 0.1, "residual": False},
        # log-probability of one token: the weights are read once
        {"name": "loss, one token", "op": "loss", "tokens": 1, "vocab": 131072, "dim": 4096, "type": "bfloat16", "out": "none"},
        # fp32 training at odd sizes
        {"name": "loss and gradients, odd, fp32", "op": "loss", "tokens": 513, "vocab": 10007, "dim": 1000, "type": "float32", "out": "float32"},
        # 16-bit activations and weights, fp32 weight gradient for the fp32 steps
        {"name": "loss and gradients, fp32 out", "op": "loss", "tokens": 2048, "vocab": 32000, "dim": 2048, "type": "bfloat16", "out": "float32"},
        # the largest: a batch against a large vocabulary, fp16 gradients for the mixed-precision step
        {"name": "loss and gradients, large", "op": "loss", "tokens": 4096, "vocab": 131072, "dim": 4096, "type": "float16", "out": "float16"},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def width(lo, hi):     # most models' widths are multiples of 64; some are not
        d = spread(lo, hi)
        return d if rng.random() < 0.4 else max(64, d // 64 * 64)

    op = rng.choice(["lookup", "table_gradient", "dropout", "loss", "loss"])
    kind = rng.choice(sorted(TYPES))
    if op == "lookup":
        return {"op": op, "tokens": spread(1, 32768), "vocab": spread(1000, 131072), "dim": width(64, 4096), "type": kind,
                "p": rng.choice([0.0, 0.1, 0.25])}
    if op == "table_gradient":
        add = rng.random() < 0.3
        return {"op": op, "tokens": spread(1, 32768), "vocab": spread(1000, 131072), "dim": width(64, 2048), "type": kind,
                "out": "float32" if add else rng.choice(["float32", kind]), "p": rng.choice([0.0, 0.0, 0.1]), "add": add}
    if op == "dropout":
        return {"op": op, "elements": spread(1000, 16383 * 4099), "type": kind, "p": rng.choice([0.05, 0.1, 0.3, 0.5]),
                "residual": rng.random() < 0.5}
    gradients = rng.random() < 0.75
    most = 2048 if kind == "float32" else 4096
    return {"op": op, "tokens": spread(1, most), "vocab": spread(1000, 131072 if kind != "float32" else 32768), "dim": width(64, most),
            "type": kind, "out": rng.choice(["float32", kind]) if gradients else "none"}


# ---------------------------------------------------------------------------------------- the program's data ----
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, (dtype, code) = case["op"], TYPES[case["type"]]
    s = {"op": op, "case": case, "dtype": dtype, "code": code}
    if case.get("p", 0.0) > 0.0 or op == "dropout":       # {seed, seed, step, 0}: one per model, advanced once a step
        s["rng"] = torch.tensor([seed & 0x7FFFFFFF, (seed * 7919) & 0x7FFFFFFF, 3, 0], dtype=torch.int32, device="cuda")
    if op == "dropout":
        n = case["elements"]
        s["x"] = torch.randn(n, generator=g, device="cuda").to(dtype)
        s["residual"] = torch.randn(n, generator=g, device="cuda").to(dtype) if case["residual"] else None
        s["y"] = torch.empty_like(s["x"])
        return s
    n, v, d = case["tokens"], case["vocab"], case["dim"]
    # words' frequencies fall about as 1 / rank; where a word stands in the vocabulary says little of its rank
    rank = torch.exp(torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * math.log(v)).long() - 1
    ids = (rank.clamp(0, v - 1) * 40503 + seed % 1000) % v
    padded = torch.rand(n, generator=g, device="cuda") < (0.1 if n > 8 else 0.0)
    if op == "loss":
        s["target"] = torch.where(padded, torch.full_like(ids, IGNORE), ids).to(torch.int32)
        s["w"] = (torch.randn(v, d, generator=g, device="cuda") * 0.02).to(dtype)
        # normalised activations; a trained model's lean towards the word that follows, some much more than others
        x = torch.randn(n, d, generator=g, device="cuda")
        lean = torch.rand(n, 1, generator=g, device="cuda") * 10.0
        s["x"] = (x + lean * s["w"][ids].float() / (0.02 * 0.02 * d)).to(dtype)
        s["losses"] = torch.empty(n, device="cuda")
        s["loss"] = torch.empty(2, device="cuda")
        s["scale"] = 1.0 if dtype != torch.float16 else 65536.0
        if case["out"] != "none":
            s["dx"] = torch.empty_like(s["x"])
            s["dw"] = torch.empty(v, d, device="cuda", dtype=TYPES[case["out"]][0])
        return s
    s["ids"] = torch.where(padded, torch.full_like(ids, -1), ids).to(torch.int32)     # -1: padding of the batch
    s["scale"] = math.sqrt(d) if op == "lookup" else 1.0
    if op == "lookup":
        s["table"] = (torch.randn(v, d, generator=g, device="cuda") * 0.02).to(dtype)
        s["y"] = torch.empty(n, d, device="cuda", dtype=dtype)
    else:
        s["dy"] = torch.randn(n, d, generator=g, device="cuda").to(dtype)
        out = TYPES[case["out"]][0]
        s["dt"] = torch.randn(v, d, generator=g, device="cuda").to(out) if case["add"] else torch.empty(v, d, device="cuda", dtype=out)
    return s


# ------------------------------------------------------------------------------------------------- one pass ----
def run(s):
    if own:
        return call(s)
    return {"lookup": plain_lookup, "table_gradient": plain_table_gradient, "dropout": plain_dropout, "loss": plain_loss}[s["op"]](s)


# -------------------------------------------------------------------------------------------- the plain forms ----
def kept(n, p, site, rng):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011): block b of eight elements has the counter (b, b >> 32, site,
    step) and the key (seed, seed); its four words give sixteen bits to each element, low halves first.  An element is
    kept where its bits reach 65536 p.  The truth values, and what a kept element is multiplied by."""
    border = int(math.floor(p * 65536.0 + 0.5))
    mask = 0xFFFFFFFF
    b = torch.arange((n + 7) // 8, device=rng.device, dtype=torch.int64)
    key = rng.to(torch.int64) & mask
    k0, k1 = key[0], key[1]
    c0, c1, c2, c3 = b & mask, b >> 32, torch.full_like(b, site), key[2].expand_as(b)
    for _ in range(10):
        a, e = c0 * 0xD2511F53, c2 * 0xCD9E8D57       # (their 64 bits: overflow wraps)
        c0, c1, c2, c3 = ((e >> 32) & mask) ^ c1 ^ k0, e & mask, ((a >> 32) & mask) ^ c3 ^ k1, a & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    words = torch.stack([c0, c1, c2, c3], 1)
    bits = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n]
    return bits >= border, 65536.0 / (65536 - border) if border < 65536 else 0.0


def plain_lookup(s):
    c = s["case"]
    ids = s["ids"].long()
    fine = (ids >= 0) & (ids < c["vocab"])
    y = s["table"][ids.clamp(0, c["vocab"] - 1)].float() * s["scale"]
    y = torch.where(fine[:, None], y, torch.zeros_like(y))
    if c["p"] > 0.0:
        keep, by = kept(y.numel(), c["p"], 0, s["rng"])
        y = torch.where(keep.view_as(y), y * by, torch.zeros_like(y))
    return y.to(s["dtype"])


def plain_table_gradient(s):
    c = s["case"]
    ids = s["ids"].long()
    fine = (ids >= 0) & (ids < c["vocab"])
    dy = s["dy"].float()
    if c["p"] > 0.0:
        keep, by = kept(dy.numel(), c["p"], 0, s["rng"])
        dy = torch.where(keep.view_as(dy), dy * by, torch.zeros_like(dy))
    total = torch.zeros(c["vocab"], c["dim"], device=dy.device).index_add_(0, ids[fine], dy[fine]) * s["scale"]
    if c["add"]:
        s["dt"].add_(total)
        return s["dt"]
    return total.to(s["dt"].dtype)


def plain_dropout(s):
    c = s["case"]
    x = s["x"].float()
    keep, by = kept(x.numel(), c["p"], 5, s["rng"])
    y = torch.where(keep, x * by, torch.zeros_like(x))
    if c["residual"]:
        y = y + s["residual"].float()
    return y.to(s["dtype"])


def plain_loss(s):
    c = s["case"]
    target = s["target"].long()
    fine = target != IGNORE
    at = target.clamp(min=0)[:, None]
    x, w = s["x"].float(), s["w"].float()
    logits = x @ w.t()
    top = logits.max(1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    losses = torch.where(fine, (torch.log(total) + top - logits.gather(1, at))[:, 0], torch.zeros_like(total[:, 0]))
    count = fine.sum()
    loss = losses.double().sum() / count.clamp(min=1)
    out = {"losses": losses, "loss": loss.float(), "count": count.float()}
    if c["out"] != "none":
        p_at = torch.exp(logits.gather(1, at) - top) / total
        ds = e.div_(total)
        ds.scatter_(1, at, p_at - 1.0)
        ds *= torch.where(fine, s["scale"] / count.clamp(min=1), torch.zeros_like(losses))[:, None]
        out["dx"] = (ds @ w).to(s["dtype"])
        out["dw"] = (ds.t() @ x).to(s["dw"].dtype)
    return out


# ------------------------------------------------------------------------------------------- the library's calls ----
_library = {}


def library():
    """The library, its device handle, and a queue handle for torch's current stream."""
    if not _library:
        from __graft_entry__ import load_package
        lib = load_package().load_library()
        _library.update(lib=lib, device=lib.create_metal_device(), queues={})
    stream = torch.cuda.current_stream().cuda_stream
    queue = _library["queues"].get(stream)
    if queue is None:
        queue = _library["lib"].gm_command_queue_for_stream(_library["device"], ctypes.c_void_p(stream))
        _library["queues"][stream] = queue
    return _library["lib"], _library["device"], queue


def workspace(s, size):
    """The call's workspace, which a program keeps for as long as its sizes stay."""
    if "workspace" not in s:
        s["workspace"] = torch.empty(max(256, size()), dtype=torch.uint8, device="cuda")
    return s["workspace"].data_ptr(), s["workspace"].numel()


def call(s):
    lib, device, queue = library()
    c, op = s["case"], s["op"]
    if op == "dropout":
        rc = lib.execute_dropout(device, queue, s["x"].data_ptr(), s["residual"].data_ptr() if c["residual"] else 0, s["y"].data_ptr(),
                                 c["elements"], s["code"], c["p"], s["rng"].data_ptr(), 5)
        out = s["y"]
    elif op == "lookup":
        rc = lib.execute_embedding_lookup(device, queue, s["table"].data_ptr(), s["ids"].data_ptr(), s["y"].data_ptr(), c["tokens"],
                                          c["vocab"], c["dim"], c["dim"], c["dim"], s["code"], s["scale"], c["p"],
                                          s["rng"].data_ptr() if c["p"] > 0.0 else 0, 0)
        out = s["y"]
    elif op == "table_gradient":
        space, size = workspace(s, lambda: lib.gm_embedding_gradient_workspace(c["tokens"], c["vocab"], c["dim"]))
        rc = lib.execute_embedding_gradient(device, queue, s["dy"].data_ptr(), s["ids"].data_ptr(), s["dt"].data_ptr(), c["tokens"],
                                            c["vocab"], c["dim"], c["dim"], c["dim"], s["code"], TYPES[c["out"]][1], s["scale"], -1,
                                            int(c["add"]), c["p"], s["rng"].data_ptr() if c["p"] > 0.0 else 0, 0, space, size)
        out = s["dt"]
    else:
        grads = c["out"] != "none"
        code = TYPES[c["out"]][1] if grads else s["code"]
        space, size = workspace(s, lambda: lib.gm_linear_cross_entropy_workspace(c["tokens"], c["vocab"], c["dim"], s["w"].data_ptr(),
                                                                                  c["dim"], s["code"], code, int(grads)))
        rc = lib.execute_linear_cross_entropy(device, queue, s["x"].data_ptr(), s["w"].data_ptr(), s["target"].data_ptr(),
                                              s["losses"].data_ptr(), s["loss"].data_ptr(), s["dx"].data_ptr() if grads else 0,
                                              s["dw"].data_ptr() if grads else 0, c["tokens"], c["vocab"], c["dim"], c["dim"], c["dim"],
                                              c["dim"], c["dim"], s["code"], code, IGNORE, 1, s["scale"], 0, 0, space, size)
        out = {"losses": s["losses"], "loss": s["loss"][0], "count": s["loss"][1]}
        if grads:
            out.update(dx=s["dx"], dw=s["dw"])
    if rc != 0:
        raise RuntimeError("%s: code %d: %s" % (op, rc, lib.gm_last_error().decode()))
    return out


# ------------------------------------------------------------------------------------------ what a pass cannot do without ----
def work(case):
    size = {"float32": 4, "float16": 2, "bfloat16": 2, "none": 0}
    b, op = size[case["type"]], case["op"]
    if op == "dropout":
        n = case["elements"]
        return {"bytes": n * b * (3 if case["residual"] else 2), "flops": 2 * n}
    n, v, d = case["tokens"], case["vocab"], case["dim"]
    if op == "lookup":
        return {"bytes": 2 * n * d * b + 4 * n, "flops": n * d}
    o = size[case["out"]]
    if op == "table_gradient":
        rows = min(n, v)
        return {"bytes": n * d * b + 4 * n + (2 * rows if case["add"] else v) * d * o, "flops": n * d}
    if case["out"] == "none":
        return {"bytes": (n + v) * d * b + 8 * n, "flops": 2 * n * v * d}
    return {"bytes": (2 * n + v) * d * b + v * d * o + 8 * n, "flops": 6 * n * v * d}


# ------------------------------------------------------------------------------------------------ in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]

    def halves(a, b):     # the product of two words as (high word, low word), by sixteen-bit digits
        a1, a0, b1, b0 = a >> 16, a & 0xFFFF, b >> 16, b & 0xFFFF
        low, mid1, mid2, high = a0 * b0, a1 * b0, a0 * b1, a1 * b1
        mid = (low >> 16) + (mid1 & 0xFFFF) + (mid2 & 0xFFFF)
        return high + (mid1 >> 16) + (mid2 >> 16) + (mid >> 16), ((mid & 0xFFFF) << 16) | (low & 0xFFFF)

    def factor(n, site):
        p, state = case.get("p", 0.0), [int(x) & 0xFFFFFFFF for x in s["rng"].tolist()]
        border = int(math.floor(p * 65536.0 + 0.5))
        block = torch.arange(-(-n // 8), device="cuda", dtype=torch.int64)
        x = [block % (1 << 32), block // (1 << 32), torch.zeros_like(block) + site, torch.zeros_like(block) + state[2]]
        for r in range(10):
            k = [(state[0] + r * 0x9E3779B9) % (1 << 32), (state[1] + r * 0xBB67AE85) % (1 << 32)]
            h0, l0 = halves(x[0], 0xD2511F53)
            h1, l1 = halves(x[2], 0xCD9E8D57)
            x = [h1 ^ x[1] ^ k[0], l1, h0 ^ x[3] ^ k[1], l0]
        bits = torch.empty(block.numel(), 8, device="cuda", dtype=torch.int64)
        for j in range(8):
            bits[:, j] = (x[j // 2] // (65536 if j % 2 else 1)) % 65536
        return (bits.view(-1)[:n] >= border).double() * (65536.0 / max(1, 65536 - border))

    if op == "dropout":
        y = s["x"].double() * factor(case["elements"], 5)
        return y + s["residual"].double() if case["residual"] else y
    n, v, d = case["tokens"], case["vocab"], case["dim"]
    if op == "lookup":
        y = torch.zeros(n, d, device="cuda", dtype=torch.float64)
        for i in range(0, n, 4096):
            ids = s["ids"][i:i + 4096].long()
            y[i:i + 4096] = s["table"].index_select(0, ids.remainder(v)).double() * (s["scale"] * (ids >= 0).double()[:, None])
        return y * factor(n * d, 0).view(n, d) if case["p"] > 0.0 else y
    if op == "table_gradient":
        dy = s["dy"].double()
        if case["p"] > 0.0:
            dy *= factor(n * d, 0).view(n, d)
        ids = s["ids"].long()
        dy[ids < 0] = 0.0
        total = s["dt"].double() if case["add"] else torch.zeros(v, d, device="cuda", dtype=torch.float64)
        return total.index_put_((ids.clamp(min=0),), dy * s["scale"], accumulate=True)
    grads = case["out"] != "none"
    w = s["w"].double()
    target = s["target"].long()
    count = int((target >= 0).sum())
    losses = torch.zeros(n, device="cuda", dtype=torch.float64)
    dx = torch.zeros(n, d, device="cuda", dtype=torch.float64) if grads else None
    dw = torch.zeros(v, d, device="cuda", dtype=torch.float64) if grads else None
    for i in range(0, n, 1024):
        rows = torch.nonzero(target[i:i + 1024] >= 0)[:, 0] + i
        if rows.numel() == 0:
            continue
        x, t = s["x"][rows].double(), target[rows]
        logits = x @ w.t()
        lse = torch.logsumexp(logits, 1)
        right = logits[torch.arange(rows.numel(), device="cuda"), t]
        losses[rows] = lse - right
        if grads:
            p = torch.exp(logits - lse[:, None])
            p[torch.arange(rows.numel(), device="cuda"), t] = torch.expm1(right - lse)
            p *= s["scale"] / count
            dx[rows] = p @ w
            dw += p.t().contiguous() @ x
    out = {"losses": losses, "loss": losses.sum() / max(1, count), "count": torch.tensor(float(count), device="cuda", dtype=torch.float64)}
    if grads:
        out.update(dx=dx, dw=dw)
    return out
