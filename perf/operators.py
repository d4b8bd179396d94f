"""The work the operators of a learned decoder of rendered images are timed on: cross attention
to an encoder's states, group norm with an activation (channels last) and embedding lookup with
its gradient by sorted tokens.

listed() names the cases, draw() makes more of the same ranges, prepare() makes a case's inputs
on the GPU from a seed, run() is one pass, work() the bytes and operations a pass needs at least,
and exact() the same results in 64 bits from the operators' definitions. With own set, run()
calls the package's operators; otherwise it computes them from elementary torch operations in
32 bits, rounded once at the end.
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
EPS = 1e-5


def _decoder():
    from __graft_entry__ import load_package
    load_package()
    from tdgs_amd import decoder
    return decoder


def listed():
    return [
        # serving one query token (a camera's) against a short set of states: all latency
        {"name": "attend_one_token", "what": "attend", "grad": False, "dtype": "bfloat16", "b": 1, "kvb": 1, "lq": 1,
         "lk": 64, "h": 4, "hk": 4, "d": 64, "layout": "blhd", "mask": "none"},
        # serving eight query tokens of eight photographs, each over a long cache of image
        # tokens of its own length, four query heads to a key head
        {"name": "attend_long_cache", "what": "attend", "grad": False, "dtype": "bfloat16", "b": 8, "kvb": 8, "lq": 1,
         "lk": 20011, "h": 16, "hk": 4, "d": 128, "layout": "bhld", "mask": "lengths"},
        # the pixels of two 1/8 scale feature images asking a short, padded token sequence
        {"name": "attend_pixels_short", "what": "attend", "grad": False, "dtype": "float16", "b": 2, "kvb": 2,
         "lq": 17115, "lk": 93, "h": 8, "hk": 8, "d": 40, "layout": "fused", "mask": "lengths"},
        # a full HD image's 1/8 scale features asking every patch of a large reference photograph
        {"name": "attend_pixels_large", "what": "attend", "grad": False, "dtype": "bfloat16", "b": 1, "kvb": 1,
         "lq": 32400, "lk": 4096, "h": 16, "hk": 16, "d": 64, "layout": "blhd", "mask": "none"},
        # training in 32 bits on crops of odd sizes, keys masked one by one, one photograph without any
        {"name": "attend_train_masked", "what": "attend", "grad": True, "dtype": "float32", "b": 3, "kvb": 3,
         "lq": 2501, "lk": 777, "h": 8, "hk": 2, "d": 64, "layout": "blhd", "mask": "keys"},
        # training on two full HD images whose pixels ask one shared set of states
        {"name": "attend_train_large", "what": "attend", "grad": True, "dtype": "bfloat16", "b": 2, "kvb": 1,
         "lq": 32400, "lk": 1024, "h": 8, "hk": 8, "d": 64, "layout": "blhd", "mask": "none"},
        # the innermost 8 x 8 feature image of one small decoder pass: all latency
        {"name": "norm_8x8", "what": "norm", "grad": False, "dtype": "float32", "n": 1, "p": 64, "c": 128,
         "groups": 32, "act": "silu"},
        # the half scale features of a full HD image on their way to the output
        {"name": "norm_960x540", "what": "norm", "grad": False, "dtype": "bfloat16", "n": 1, "p": 518400, "c": 128,
         "groups": 32, "act": "silu"},
        # training on three quarter scale feature images of an odd size
        {"name": "norm_train_ragged", "what": "norm", "grad": True, "dtype": "float32", "n": 3, "p": 33565, "c": 96,
         "groups": 8, "act": "gelu"},
        # the embedding tokens of a few photographs, and their gradient
        {"name": "embed_train_small", "what": "embed", "grad": True, "dtype": "float32", "t": 96, "v": 1000, "d": 64,
         "index": "int64"},
        # a million Gaussians' degree 3 colours from a codebook, and the codebook's gradient
        {"name": "embed_train_codebook", "what": "embed", "grad": True, "dtype": "float32", "t": 1000000, "v": 8192,
         "d": 48, "index": "int32"},
        # wide rows of a large table for a batch of token sequences, and the table's gradient
        {"name": "embed_train_wide", "what": "embed", "grad": True, "dtype": "bfloat16", "t": 65537, "v": 100003,
         "d": 512, "index": "int64"},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    what = rng.choice(["attend", "attend", "attend", "attend", "norm", "norm", "embed", "embed"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if what == "attend":
        while True:
            b = rng.choice([1, 1, 2, 3, 4, 8])
            hk = rng.choice([1, 2, 4, 8])
            case = {"what": "attend", "grad": rng.random() < 0.5, "dtype": dtype, "b": b,
                    "kvb": rng.choice([b, b, 1]), "lq": rng.choice([1, _log_uniform(rng, 2, 33000)]),
                    "lk": _log_uniform(rng, 1, 20000), "h": hk * rng.choice([1, 1, 2, 4]), "hk": hk,
                    "d": rng.choice([16, 32, 40, 64, 64, 80, 128, rng.randint(8, 128)]),
                    "layout": rng.choice(["blhd", "bhld", "fused"]),
                    "mask": rng.choice(["none", "lengths", "keys"])}
            if case["grad"] and case["lq"] == 1:
                continue
            scores = case["b"] * case["h"] * case["lq"] * case["lk"]
            # at most the largest listed cases' work and the plain form's score matrices
            rate = 8 if dtype == "float32" else 1
            if rate * work(case)["flops"] <= 4.5e11 and scores <= 2e9:
                return case
    if what == "norm":
        while True:
            groups = rng.choice([1, 4, 8, 16, 32])
            case = {"what": "norm", "grad": rng.random() < 0.5, "dtype": dtype, "n": rng.choice([1, 1, 2, 3, 8]),
                    "p": _log_uniform(rng, 1, 518400), "c": groups * rng.choice([1, 3, 4, 8, 10, 16]),
                    "groups": groups, "act": rng.choice(["identity", "silu", "silu", "gelu"])}
            if case["n"] * case["p"] * case["c"] <= 518400 * 128:
                return case
    while True:
        case = {"what": "embed", "grad": rng.random() < 0.7, "dtype": dtype, "t": _log_uniform(rng, 1, 1000000),
                "v": _log_uniform(rng, 2, 100003), "d": rng.choice([1, 3, 16, 27, 48, 64, 256, 512]),
                "index": rng.choice(["int32", "int64"])}
        if max(case["t"], case["v"]) * case["d"] <= 1000000 * 48:
            return case


# ------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1_000_003 * (int(seed) + 1))
    return g


def _attend_inputs(case, seed):
    """q, k, v, the keys' lengths or mask, and the output's gradient. Keys that are not allowed hold
    what uninitialised memory may hold: NaN."""
    g = _generator(seed)
    t = TYPES[case["dtype"]]
    b, kvb, lq, lk, h, hk, d = (case[x] for x in ("b", "kvb", "lq", "lk", "h", "hk", "d"))

    def heads(batch, length, n):
        if case["layout"] == "bhld":
            return torch.randn((batch, n, length, d), generator=g, device=DEV).to(t).transpose(1, 2)
        return torch.randn((batch, length, n, d), generator=g, device=DEV).to(t)

    q = 1.5 * heads(b, lq, h)
    if case["layout"] == "fused":   # keys and values of one projection
        kv = torch.randn((kvb, lk, 2, hk, d), generator=g, device=DEV).to(t)
        k, v = kv[:, :, 0], kv[:, :, 1]
    else:
        k, v = heads(kvb, lk, hk), heads(kvb, lk, hk)
    lengths = mask = None
    if case["mask"] == "lengths":
        lengths = torch.randint((lk + 1) // 2, lk + 1, (kvb,), generator=g, device=DEV).to(torch.int32)
        keep = torch.arange(lk, device=DEV)[None, :] < lengths[:, None]
    elif case["mask"] == "keys":
        mask = torch.rand((kvb, lk), generator=g, device=DEV) < 0.7
        mask[0] = False   # nothing to look at
        if kvb == 1:
            mask[0, ::2] = True
        keep = mask
    if case["mask"] != "none":
        k.masked_fill_(~keep[:, :, None, None], float("nan"))
        v.masked_fill_(~keep[:, :, None, None], float("nan"))
    dout = heads(b, lq, h) if case["grad"] else None
    return q, k, v, lengths, mask, dout


def _norm_inputs(case, seed):
    """Features with a mean and a spread per channel, the affine parameters, and the output's gradient."""
    g = _generator(seed)
    t = TYPES[case["dtype"]]
    n, p, c = case["n"], case["p"], case["c"]
    mean = torch.randn((c,), generator=g, device=DEV)
    spread = torch.exp(0.5 * torch.randn((c,), generator=g, device=DEV))
    x = (torch.randn((n, p, c), generator=g, device=DEV) * spread + mean).to(t)
    weight = 1 + 0.2 * torch.randn((c,), generator=g, device=DEV)
    bias = 0.2 * torch.randn((c,), generator=g, device=DEV)
    dout = torch.randn((n, p, c), generator=g, device=DEV).to(t) if case["grad"] else None
    return x, weight, bias, dout


def _embed_inputs(case, seed):
    """A table, tokens whose frequency falls with their rank (ranks in any order), and the rows' gradient."""
    g = _generator(seed)
    t = TYPES[case["dtype"]]
    table = torch.randn((case["v"], case["d"]), generator=g, device=DEV).to(t)
    rank = torch.rand((case["t"],), generator=g, device=DEV, dtype=torch.float64)
    rank = torch.clamp(torch.exp(rank * math.log(case["v"] + 1)).long() - 1, 0, case["v"] - 1)
    tokens = torch.randperm(case["v"], generator=g, device=DEV)[rank].to(getattr(torch, case["index"]))
    dout = torch.randn((case["t"], case["d"]), generator=g, device=DEV).to(t) if case["grad"] else None
    return table, tokens, dout


def _embed_scale(case):
    return math.sqrt(case["d"])


def prepare(case, seed):
    state = {"case": case}
    if case["what"] == "attend":
        q, k, v, lengths, mask, dout = _attend_inputs(case, seed)
        state.update(q=q, k=k, v=v, lengths=lengths, mask=mask, dout=dout)
        if own:
            dec = _decoder()
            state.update(out=torch.empty_like(q), temp=dec.cross_attention_temp(q, k, grad=case["grad"]))
            if case["grad"]:
                state.update(lse=torch.empty((case["b"], case["h"], case["lq"]), device=DEV), dq=torch.empty_like(q),
                             dk=torch.empty(k.shape, dtype=k.dtype, device=DEV),
                             dv=torch.empty(v.shape, dtype=v.dtype, device=DEV))
    elif case["what"] == "norm":
        x, weight, bias, dout = _norm_inputs(case, seed)
        state.update(x=x, weight=weight, bias=bias, dout=dout)
        if own:
            dec = _decoder()
            state.update(out=torch.empty_like(x), temp=dec.group_norm_temp(x, case["groups"], grad=case["grad"]))
            if case["grad"]:
                state.update(stats=torch.empty((case["n"], case["groups"], 2), device=DEV), dx=torch.empty_like(x),
                             dweight=torch.empty_like(weight), dbias=torch.empty_like(bias))
    else:
        table, tokens, dout = _embed_inputs(case, seed)
        state.update(table=table, tokens=tokens, dout=dout)
        if own:
            dec = _decoder()
            state.update(out=torch.empty((case["t"], case["d"]), dtype=table.dtype, device=DEV))
            if case["grad"]:
                state.update(dtable=torch.empty_like(table), temp=dec.embedding_temp(table, tokens))
    if own:
        state["decoder"] = dec
    return state


# ------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------

def _keep(case, lengths, mask):
    if lengths is not None:
        return torch.arange(case["lk"], device=DEV)[None, :] < lengths[:, None]
    return mask


def _attend_plain(s):
    case = s["case"]
    t, group = TYPES[case["dtype"]], case["h"] // case["hk"]
    scale = 1 / math.sqrt(case["d"])
    q, k, v = (s[x].float().transpose(1, 2) for x in ("q", "k", "v"))   # (b, heads, length, d)
    keep = _keep(case, s["lengths"], s["mask"])
    if keep is not None:
        k = torch.where(keep[:, None, :, None], k, 0.0)
        v = torch.where(keep[:, None, :, None], v, 0.0)
    shape = (case["b"], case["hk"], group, case["lk"], case["d"])
    kr = k[:, :, None].expand(shape).reshape(case["b"], case["h"], case["lk"], case["d"])
    vr = v[:, :, None].expand(shape).reshape(case["b"], case["h"], case["lk"], case["d"])
    p = torch.matmul(q, kr.transpose(2, 3)).mul_(scale)
    if keep is not None:
        p.masked_fill_(~keep[:, None, None, :], float("-inf"))
    top = p.amax(dim=-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    p.div_(torch.where(total == 0, 1.0, total))
    out = torch.matmul(p, vr)
    if not case["grad"]:
        return out.transpose(1, 2).to(t)
    do = s["dout"].float().transpose(1, 2)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, vr.transpose(2, 3))
    ds.sub_((do * out).sum(dim=-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, kr)
    dk = torch.matmul(ds.transpose(2, 3), q)
    dk = dk.reshape(shape).sum(dim=2)
    dv = dv.reshape(shape).sum(dim=2)
    if case["kvb"] < case["b"]:
        dk, dv = dk.sum(dim=0, keepdim=True), dv.sum(dim=0, keepdim=True)
    return tuple(x.transpose(1, 2).to(t) for x in (out, dq, dk, dv))


def _act_plain(z, act):
    """act(z) and its derivative."""
    if act == "identity":
        return z, torch.ones_like(z)
    if act == "silu":
        sg = 1 / (1 + torch.exp(-z))
        return z * sg, sg * (1 + z * (1 - sg))
    cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _norm_plain(s):
    case = s["case"]
    t = TYPES[case["dtype"]]
    shape = (case["n"], case["p"], case["groups"], case["c"] // case["groups"])
    x = s["x"].float().reshape(shape)
    w, b = (s[k].reshape(1, 1, *shape[2:]) for k in ("weight", "bias"))
    xhat = x - x.mean(dim=(1, 3), keepdim=True)
    r = 1 / torch.sqrt((xhat * xhat).mean(dim=(1, 3), keepdim=True) + EPS)
    xhat = xhat * r
    y, slope = _act_plain(xhat * w + b, case["act"])
    out = y.reshape(s["x"].shape).to(t)
    if not case["grad"]:
        return out
    e = s["dout"].float().reshape(shape) * slope
    db = e.sum(dim=(0, 1)).reshape(-1)
    dw = (e * xhat).sum(dim=(0, 1)).reshape(-1)
    e = e * w
    dx = r * (e - e.mean(dim=(1, 3), keepdim=True) - xhat * (e * xhat).mean(dim=(1, 3), keepdim=True))
    return out, dx.reshape(s["x"].shape).to(t), dw, db


def _embed_plain(s):
    case = s["case"]
    t, scale = TYPES[case["dtype"]], _embed_scale(case)
    tokens = s["tokens"].long()
    out = (s["table"][tokens].float() * scale).to(t)
    if not case["grad"]:
        return out
    dtable = torch.zeros((case["v"], case["d"]), device=DEV)
    dtable.index_add_(0, tokens, s["dout"].float())
    return out, (dtable * scale).to(t)


def run(state):
    case = state["case"]
    if not own:
        return {"attend": _attend_plain, "norm": _norm_plain, "embed": _embed_plain}[case["what"]](state)
    dec = state["decoder"]
    if case["what"] == "attend":
        keys = {"kv_lengths": state["lengths"], "kv_mask": state["mask"]}
        if not case["grad"]:
            dec.cross_attention_(state["out"], state["q"], state["k"], state["v"], temp=state["temp"], **keys)
            return state["out"]
        dec.cross_attention_(state["out"], state["q"], state["k"], state["v"], lse=state["lse"], temp=state["temp"],
                             **keys)
        dec.cross_attention_grad_(state["dq"], state["dk"], state["dv"], state["dout"], state["out"], state["lse"],
                                  state["q"], state["k"], state["v"], temp=state["temp"], **keys)
        return state["out"], state["dq"], state["dk"], state["dv"]
    if case["what"] == "norm":
        if not case["grad"]:
            dec.group_norm_(state["out"], state["x"], case["groups"], state["weight"], state["bias"], eps=EPS,
                            activation=case["act"], temp=state["temp"])
            return state["out"]
        dec.group_norm_(state["out"], state["x"], case["groups"], state["weight"], state["bias"], eps=EPS,
                        activation=case["act"], stats=state["stats"], temp=state["temp"])
        dec.group_norm_grad_(state["dx"], state["dweight"], state["dbias"], state["dout"], state["x"], state["stats"],
                             case["groups"], state["weight"], state["bias"], activation=case["act"],
                             temp=state["temp"])
        return state["out"], state["dx"], state["dweight"], state["dbias"]
    scale = _embed_scale(case)
    dec.embedding_lookup_(state["out"], state["table"], state["tokens"], scale=scale)
    if not case["grad"]:
        return state["out"]
    dec.embedding_grad_(state["dtable"], state["dout"], state["tokens"], scale=scale, temp=state["temp"])
    return state["out"], state["dtable"]


# ------------------------------------------------------------------------------------
# The least a pass needs
# ------------------------------------------------------------------------------------

def work(case):
    e = BYTES[case["dtype"]]
    if case["what"] == "attend":
        rows, keys = case["b"] * case["lq"] * case["h"], case["kvb"] * case["lk"] * case["hk"]
        scores = rows * case["lk"]
        if not case["grad"]:
            return {"bytes": e * case["d"] * (2 * rows + 2 * keys), "flops": 4 * scores * case["d"]}
        # q and its gradient, the output and its gradient; k, v and theirs. Forward 2 products, backward 5
        return {"bytes": e * case["d"] * (4 * rows + 4 * keys), "flops": 14 * scores * case["d"]}
    if case["what"] == "norm":
        n = case["n"] * case["p"] * case["c"]
        if not case["grad"]:
            return {"bytes": e * 2 * n + 8 * case["c"], "flops": 10 * n}
        return {"bytes": e * 4 * n + 16 * case["c"], "flops": 30 * n}
    rows, index = case["t"] * case["d"], 4 if case["index"] == "int32" else 8
    bytes_ = e * (rows + min(case["t"], case["v"]) * case["d"]) + index * case["t"]
    if case["grad"]:
        bytes_ += e * (rows + case["v"] * case["d"])
    return {"bytes": bytes_, "flops": rows * (2 if case["grad"] else 1)}


# ------------------------------------------------------------------------------------
# The same results in 64 bits
# ------------------------------------------------------------------------------------

def _exact_attend(case, seed):
    q, k, v, lengths, mask, dout = _attend_inputs(case, seed)
    group, scale = case["h"] // case["hk"], case["d"] ** -0.5
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    grads = [torch.zeros(x.shape, dtype=torch.float64, device=DEV) for x in (q, k, v)] if case["grad"] else None
    for b in range(case["b"]):
        kb = b if case["kvb"] > 1 else 0
        allowed = torch.arange(case["lk"], device=DEV)
        if lengths is not None:
            allowed = allowed[:int(lengths[kb])]
        if mask is not None:
            allowed = torch.nonzero(mask[kb]).flatten()
        if allowed.numel() == 0:
            continue
        for h in range(case["h"]):
            hk = h // group
            x = [q[b, :, h].double(), k[kb, allowed, hk].double(), v[kb, allowed, hk].double()]
            for y in x:
                y.requires_grad_(case["grad"])
            o = torch.softmax(x[0] @ x[1].T * scale, dim=1) @ x[2]
            out[b, :, h] = o.detach()
            if case["grad"]:
                gq, gk, gv = torch.autograd.grad(o, x, dout[b, :, h].double())
                grads[0][b, :, h] = gq
                grads[1][kb, allowed, hk] += gk
                grads[2][kb, allowed, hk] += gv
    return (out, *grads) if case["grad"] else out


def _exact_norm(case, seed):
    x, weight, bias, dout = _norm_inputs(case, seed)
    leaves = [y.double().requires_grad_(case["grad"]) for y in (x, weight, bias)]
    # groups first: (n, groups, p, channels of a group)
    y = leaves[0].unflatten(2, (case["groups"], -1)).permute(0, 2, 1, 3)
    var, mean = torch.var_mean(y, dim=(2, 3), unbiased=False, keepdim=True)
    y = ((y - mean) * torch.rsqrt(var + EPS)).permute(0, 2, 1, 3).flatten(2)
    y = y * leaves[1] + leaves[2]
    act = {"identity": lambda z: z, "silu": lambda z: z * torch.sigmoid(z),
           "gelu": lambda z: 0.5 * z * torch.erfc(-z / math.sqrt(2))}[case["act"]]
    y = act(y)
    if not case["grad"]:
        return y
    return (y.detach(), *torch.autograd.grad(y, leaves, dout.double()))


def _exact_embed(case, seed):
    table, tokens, dout = _embed_inputs(case, seed)
    scale, tokens = _embed_scale(case), tokens.long()
    out = torch.index_select(table.double(), 0, tokens) * scale
    if not case["grad"]:
        return out
    order = torch.argsort(tokens, stable=True)
    sums = torch.zeros((case["v"], case["d"]), dtype=torch.float64, device=DEV)
    sums.index_put_((tokens[order],), dout.double()[order], accumulate=True)
    return out, sums * scale


def exact(case, seed):
    return {"attend": _exact_attend, "norm": _exact_norm, "embed": _exact_embed}[case["what"]](case, seed)
