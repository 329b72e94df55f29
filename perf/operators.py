"""Cases that time the operators on rows of device tensors: table lookups with their gradient, rows sorted by group and
back with their gradients, and products of 8-bit rows with scales.

`run` computes a case in plain torch operations, or, where `own` is true, through superkmeans_amd.rowops.  `exact` computes
the same from the operators' definitions in 64 bits.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
IDS = {"u32": torch.int32, "i64": torch.int64}  # a 32-bit id is read as unsigned: -1 stands for 0xffffffff

_operators = {}  # by stream


def _own_operators():
    stream = torch._C._cuda_getCurrentRawStream(0)  # current_stream().cuda_stream, which takes as long as half a short call
    if stream not in _operators:
        from superkmeans_amd.rowops import RowOperators

        _operators[stream] = RowOperators(device=0, stream=stream)
    return _operators[stream]


# --------------------------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------------------------


def listed():
    return [
        # one decoding step of 64 sequences: their last tokens' embeddings, scaled by sqrt(d)
        dict(name="lookup_decode", op="lookup", type="bf16", ids="i64", tokens=64, rows=65536, d=4096, scale=64.0, absent=0.0),
        # a million points rebuilt from a codebook of 10,000 centroids and their assignments (the size of the benchmark)
        dict(name="lookup_codebook_1M", op="lookup", type="f32", ids="u32", tokens=1000000, rows=10000, d=1024, scale=1.0,
             absent=0.0),
        # gradient of a small codebook from one ragged batch
        dict(name="lookup_grad_small", op="lookup_grad", type="f32", out="f32", ids="u32", tokens=1021, rows=4096, d=768,
             scale=1.0, absent=0.0),
        # gradient of an embedding table from a padded training batch of text: a few ids hold much of it
        dict(name="lookup_grad_text", op="lookup_grad", type="bf16", out="f32", ids="i64", tokens=65536, rows=65536, d=1536,
             scale=1.0, absent=0.07),
        # one decoding step of 64 sequences sent to 8 of 64 experts each
        dict(name="to_groups_decode", op="to", type="bf16", tokens=64, choices=8, groups=64, d=1024, skew=0.5, dropped=0.0),
        # a long prompt sent to 2 of 8 experts, some choices dropped
        dict(name="to_groups_prompt", op="to", type="bf16", tokens=32768, choices=2, groups=8, d=4096, skew=0.5, dropped=0.03),
        # the experts' rows of a prompt brought back, weighted
        dict(name="back_prompt", op="back", type="bf16", tokens=16384, choices=8, groups=64, d=1536, skew=0.5, dropped=0.0),
        # the backward pass of sorting and bringing back, odd sizes
        dict(name="to_and_back_grad", op="grad", type="f32", tokens=10007, choices=4, groups=100, d=1000, skew=1.0,
             dropped=0.02),
        # a linear layer of 8-bit weights on a single token
        dict(name="product_token", op="product", x="bf16", out="bf16", m=1, n=4096, k=4096, groups=0, bias=False, skew=0.0,
             dropped=0.0),
        # the same layer kind on a long prompt
        dict(name="product_prompt", op="product", x="bf16", out="bf16", m=8192, n=8192, k=4096, groups=0, bias=False, skew=0.0,
             dropped=0.0),
        # the experts' layers in a decoding step: 512 rows over 64 experts
        dict(name="product_groups_decode", op="product", x="bf16", out="bf16", m=512, n=2048, k=1024, groups=64, bias=False,
             skew=0.5, dropped=0.0),
        # the experts' layers on a prompt, rows already in 8 bits
        dict(name="product_groups_prompt", op="product", x="i8", out="bf16", m=32768, n=4096, k=1536, groups=8, bias=True,
             skew=0.5, dropped=0.03),
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is spread evenly."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A row length: mostly a multiple of 8 or more, as models have them, sometimes any number."""
    n = _spread(rng, low, high)
    step = rng.choice([1, 8, 16, 64, 128, 128])
    return max(step, n // step * step)


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "to", "back", "grad", "product", "product", "product_groups"])
    kind = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op in ("lookup", "lookup_grad"):
        most = 1 << (30 if op == "lookup" else 27)
        d = _width(rng, 32, 8192)
        tokens = _spread(rng, 1, min(1 << 20, most // d))
        rows = _spread(rng, 64, min(1 << 18, (1 << 27) // d))
        case = dict(op=op, type=kind, ids=rng.choice(["u32", "i64"]), tokens=tokens, rows=rows, d=d,
                    scale=rng.choice([1.0, 0.125, math.sqrt(d)]), absent=rng.choice([0.0, 0.0, 0.1]))
        if op == "lookup_grad":
            case["out"] = rng.choice(["f32", kind])
        return case
    if op in ("to", "back", "grad"):
        d = _width(rng, 64, 8192)
        groups = _spread(rng, 2, 1024)
        choices = min(groups, rng.choice([1, 2, 4, 6, 8]))
        tokens = _spread(rng, 1, min(1 << 17, (1 << 27) // (d * choices)))
        return dict(op=op, type=kind, tokens=tokens, choices=choices, groups=groups, d=d, skew=rng.choice([0.0, 0.5, 1.0]),
                    dropped=rng.choice([0.0, 0.0, 0.05]))
    k = _width(rng, 64, 8192)
    n = _width(rng, 64, 8192)
    x, out = rng.choice(["bf16", "f16", "f32", "i8"]), rng.choice(["bf16", "f16", "f32"])
    if op == "product":
        m = _spread(rng, 1, min(16384, (1 << 37) // (n * k)))
        return dict(op="product", x=x, out=out, m=m, n=n, k=k, groups=0, bias=rng.random() < 0.3, skew=0.0, dropped=0.0)
    groups = max(1, _spread(rng, 4, 128) * 65536 // max(65536, n * k // 16))
    m = _spread(rng, 1, min(16384, (1 << 35) // (n * k)))
    return dict(op="product", x=x, out=out, m=m, n=n, k=k, groups=groups, bias=rng.random() < 0.3, skew=rng.choice([0.0, 0.5, 1.0]),
                dropped=rng.choice([0.0, 0.0, 0.05]))


# --------------------------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------------------------


def _normal(g, shape, kind, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(TYPES[kind])


def _choices(g, case):
    """The groups each token chooses, distinct, some groups more often than others; dropped choices hold -1."""
    t, e, k = case["tokens"], case["groups"], case["choices"]
    favour = torch.randn(e, generator=g, device="cuda") * case["skew"]
    chosen = (torch.randn((t, e), generator=g, device="cuda") + favour).topk(k, dim=1).indices.to(torch.int32)
    lost = torch.rand((t, k), generator=g, device="cuda") < case["dropped"]
    return torch.where(lost, torch.full_like(chosen, -1), chosen).contiguous()


def _sorted_places(choices, groups):
    """(slots, order, offsets) of the choices sorted by group, ties by their place; dropped ones behind, without a slot."""
    key = choices.reshape(-1).to(torch.int64)
    key = torch.where((key < 0) | (key >= groups), torch.full_like(key, groups), key)
    ordered, order = torch.sort(key, stable=True)
    place = torch.arange(key.numel(), device=key.device, dtype=torch.int32)
    slots = torch.empty_like(place)
    slots[order] = torch.where(ordered < groups, place, torch.full_like(place, -1))
    order = torch.where(ordered < groups, order.to(torch.int32), torch.full_like(place, -1))
    offsets = torch.searchsorted(ordered, torch.arange(groups + 1, device=key.device)).to(torch.int32)
    return slots.reshape(choices.shape), order, offsets


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    op = case["op"]
    if op in ("lookup", "lookup_grad"):
        t, rows, d = case["tokens"], case["rows"], case["d"]
        # id v comes up about 1 / (v + 1) as often as id 0, like words in text
        u = torch.rand(t, generator=g, device="cuda", dtype=torch.float64)
        at = (torch.exp(u * math.log(rows + 1)) - 1).to(torch.int64).clamp(0, rows - 1)
        absent = torch.rand(t, generator=g, device="cuda") < case["absent"]
        s["at"] = torch.where(absent, torch.full_like(at, -1), at).to(IDS[case["ids"]])
        if op == "lookup":
            s["table"] = _normal(g, (rows, d), case["type"], 0.02)
            s["result"] = torch.empty((t, d), device="cuda", dtype=TYPES[case["type"]])
        else:
            s["given"] = _normal(g, (t, d), case["type"], 0.1)
            s["result"] = torch.empty((rows, d), device="cuda", dtype=TYPES[case["out"]])
    elif op in ("to", "back", "grad"):
        t, k, e, d = case["tokens"], case["choices"], case["groups"], case["d"]
        kind = TYPES[case["type"]]
        chosen = _choices(g, case)
        s["slots"], s["order"], s["offsets"] = (torch.empty(n, device="cuda", dtype=torch.int32) for n in ((t, k), (t * k,), (e + 1,)))
        if op == "to":
            s["chosen"] = chosen
            s["x"] = _normal(g, (t, d), case["type"])
            s["result"] = torch.zeros((t * k, d), device="cuda", dtype=kind)  # rows behind the last group stay as they are
        else:
            s["slots"], s["order"], s["offsets"] = _sorted_places(chosen, e)
            s["weights"] = torch.rand((t, k), generator=g, device="cuda").softmax(dim=1)
            s["given_rows"] = _normal(g, (t * k, d), case["type"])
            s["result"] = torch.empty((t, d), device="cuda", dtype=kind)
            if op == "grad":
                s["given"] = _normal(g, (t, d), case["type"])
                s["given_sorted"] = _normal(g, (t * k, d), case["type"])
                s["result_rows"] = torch.zeros((t * k, d), device="cuda", dtype=kind)
                s["result_weights"] = torch.empty((t, k), device="cuda")
    else:
        m, n, k, e = case["m"], case["n"], case["k"], case["groups"]
        s["w"] = torch.randint(-127, 128, (max(1, e), n, k), generator=g, device="cuda", dtype=torch.int8)
        s["w_scales"] = (torch.rand((max(1, e), n), generator=g, device="cuda") + 0.5) * 1e-4
        s["bias"] = torch.randn((max(1, e), n), generator=g, device="cuda") if case["bias"] else None
        if e == 0:
            s["w"], s["w_scales"], s["bias"] = s["w"][0], s["w_scales"][0], None if s["bias"] is None else s["bias"][0]
            s["offsets"] = None
        else:
            share = (torch.randn(e, generator=g, device="cuda") * case["skew"]).softmax(0)
            group = torch.multinomial(share, m, replacement=True, generator=g)
            lost = torch.rand(m, generator=g, device="cuda") < case["dropped"]
            group = torch.where(lost, torch.full_like(group, e), group).sort().values
            s["offsets"] = torch.searchsorted(group, torch.arange(e + 1, device="cuda")).to(torch.int32)
        if case["x"] == "i8":
            s["x"] = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
            s["x_scales"] = torch.rand(m, generator=g, device="cuda") * 0.05
        else:
            # activations: a few columns are much larger than the rest
            wide = torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 8.0, 1.0)
            s["x"] = (torch.randn((m, k), generator=g, device="cuda") * wide).to(TYPES[case["x"]])
            s["q"] = torch.empty((m, k), device="cuda", dtype=torch.int8)
            s["x_scales"] = torch.empty(m, device="cuda")
        s["result"] = torch.zeros((m, n), device="cuda", dtype=TYPES[case["out"]])
    return s


# --------------------------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------------------------


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    ops = _own_operators()
    op = s["op"]
    if op == "lookup":
        return ops.lookup(s["table"], s["at"], s["result"], scale=s["scale"])
    if op == "lookup_grad":
        return ops.lookup_grad(s["given"], s["at"], s["result"], scale=s["scale"])
    if op == "to":
        ops.route(s["chosen"], s["groups"], s["slots"], s["offsets"], order=s["order"])
        ops.dispatch(s["x"], s["slots"], s["result"])
        return {"rows": s["result"], "slots": s["slots"], "order": s["order"], "offsets": s["offsets"]}
    if op == "back":
        return ops.combine(s["given_rows"], s["slots"], s["result"], weights=s["weights"])
    if op == "grad":
        ops.combine_grad(s["given"], s["given_rows"], s["slots"], s["weights"], s["result_rows"], s["result_weights"])
        ops.combine(s["given_sorted"], s["slots"], s["result"])
        return {"rows": s["result_rows"], "weights": s["result_weights"], "x": s["result"]}
    x = s["x"]
    if "q" in s:
        ops.quantize(x, s["q"], s["x_scales"])
        x = s["q"]
    return ops.product(x, s["x_scales"], s["w"], s["w_scales"], s["result"], bias=s["bias"], offsets=s["offsets"])


def _run_plain(s):
    op = s["op"]
    if op == "lookup":
        at, rows = s["at"], s["rows"]
        there = (at >= 0) & (at < rows)
        picked = s["table"][at.clamp(0, rows - 1)].float() * s["scale"]
        return torch.where(there[:, None], picked, 0.0).to(s["table"].dtype)
    if op == "lookup_grad":
        at, rows = s["at"].to(torch.int64), s["rows"]
        at = torch.where((at >= 0) & (at < rows), at, rows)
        total = torch.zeros((rows + 1, s["d"]), device=at.device)
        total.index_add_(0, at, s["given"].float())
        return (total[:rows] * s["scale"]).to(s["result"].dtype)
    if op == "to":
        slots, order, offsets = _sorted_places(s["chosen"], s["groups"])
        rows = s["x"][order.clamp(min=0).to(torch.int64) // s["choices"]]
        rows = torch.where((order >= 0)[:, None], rows, 0.0)
        return {"rows": rows, "slots": slots, "order": order, "offsets": offsets}
    if op == "back":
        return _plain_back(s["given_rows"], s["slots"], s["weights"]).to(s["given_rows"].dtype)
    if op == "grad":
        slots, kind = s["slots"], s["given"].dtype
        there = slots >= 0
        given = s["given"].float()
        picked = s["given_rows"][slots.clamp(min=0).to(torch.int64)].float()
        weights = torch.where(there, (picked * given[:, None, :]).sum(-1), 0.0)
        order = s["order"]
        source = order.clamp(min=0).to(torch.int64)
        rows = given[source // s["choices"]] * s["weights"].reshape(-1)[source][:, None]
        rows = torch.where((order >= 0)[:, None], rows, 0.0).to(kind)
        return {"rows": rows, "weights": weights, "x": _plain_back(s["given_sorted"], slots, None).to(kind)}
    x = s["x"]
    if x.dtype == torch.int8:
        q, scales = x.float(), s["x_scales"]
    else:
        most = x.abs().amax(dim=1).float()
        scales = most / 127.0
        # in 64 bits: a quotient next to the border between two whole numbers decides which of them is taken
        q = torch.round(x.double() * 127.0 / most.double()[:, None])
        q = torch.where(most[:, None] > 0, q, 0.0).float()
    w = s["w"].float()
    if s["offsets"] is None:
        y = (q @ w.t()) * scales[:, None] * s["w_scales"][None, :]
        if s["bias"] is not None:
            y = y + s["bias"]
        return y.to(s["result"].dtype)
    # rows of every group padded to the longest one's length: one batched product over all groups
    e, m, offsets = s["groups"], s["m"], s["offsets"].to(torch.int64)
    place = torch.arange(m, device=x.device)
    group = torch.searchsorted(offsets, place, right=True) - 1  # e for the rows behind the last group
    most = max(1, int((offsets[1:] - offsets[:-1]).max()))
    there = group < e
    group = group.clamp(max=e - 1)
    inside = (place - offsets[group]).clamp(0, most)  # a rest of dropped rows goes to a spare place
    inside = torch.where(there, inside, most)
    padded = torch.zeros((e, most + 1, s["k"]), device=x.device)
    padded[group, inside] = q
    y = torch.bmm(w, padded[:, :most].transpose(1, 2).contiguous())  # e x n x most
    y = y.transpose(1, 2)[group, inside.clamp(max=most - 1)] * scales[:, None] * s["w_scales"][group]
    if s["bias"] is not None:
        y = y + s["bias"][group]
    return torch.where(there[:, None], y, 0.0).to(s["result"].dtype)


def _plain_back(rows, slots, weights):
    there = (slots >= 0)[..., None]
    picked = torch.where(there, rows[slots.clamp(min=0).to(torch.int64)].float(), 0.0)
    return (picked if weights is None else picked * weights[..., None]).sum(dim=1)


# --------------------------------------------------------------------------------------------------------------------
# what a pass has to read, write and compute
# --------------------------------------------------------------------------------------------------------------------

SIZE = {"f32": 4, "f16": 2, "bf16": 2, "u32": 4, "i64": 8, "i8": 1}


def work(case):
    op = case["op"]
    if op in ("lookup", "lookup_grad"):
        t, rows, d = case["tokens"], case["rows"], case["d"]
        ids = t * SIZE[case["ids"]]
        if op == "lookup":
            return {"bytes": ids + (min(t, rows) + t) * d * SIZE[case["type"]], "flops": t * d}
        return {"bytes": ids + t * d * SIZE[case["type"]] + rows * d * SIZE[case["out"]], "flops": t * d}
    if op in ("to", "back", "grad"):
        t, k, d, z = case["tokens"], case["choices"], case["d"], SIZE[case["type"]]
        if op == "to":
            return {"bytes": 12 * t * k + 4 * case["groups"] + (t + t * k) * d * z, "flops": 0}
        if op == "back":
            return {"bytes": 8 * t * k + (t * k + t) * d * z, "flops": 2 * t * k * d}
        return {"bytes": 12 * t * k + (t + 2 * t * k) * d * z + (t * k + t) * d * z, "flops": 4 * t * k * d}
    m, n, k, e = case["m"], case["n"], case["k"], max(1, case["groups"])
    touched = min(e, m)
    moved = m * k * SIZE[case["x"]] + touched * n * (k + 4 + 4 * bool(case["bias"])) + m * n * SIZE[case["out"]]
    return {"bytes": moved, "flops": 2 * m * n * k}


# --------------------------------------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# --------------------------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op, f64 = case["op"], torch.float64
    if op == "lookup":
        # one row of zeros at either end of the table stands for the ids outside of it
        at = s["at"].to(torch.int64)
        at[(at < 0) | (at >= case["rows"])] = case["rows"]
        padded = torch.cat([s["table"].to(f64) * case["scale"], torch.zeros((1, case["d"]), device="cuda", dtype=f64)])
        return padded.index_select(0, at)
    if op == "lookup_grad":
        # prefix sums over the sorted tokens, taken apart at the ids' borders: no sum per id is formed step by step
        at = s["at"].to(torch.int64)
        keep = ((at >= 0) & (at < case["rows"])).nonzero()[:, 0]
        at, back = at[keep].sort(stable=True)
        given = s["given"][keep][back].to(f64)
        border = torch.searchsorted(at, torch.arange(case["rows"] + 1, device="cuda"))
        sums = torch.cat([torch.zeros((1, case["d"]), device="cuda", dtype=f64), given.cumsum(0)])
        return (sums[border[1:]] - sums[border[:-1]]) * case["scale"]
    if op == "to":
        # the place of a choice is the number of choices before it in the order (group, place)
        chosen = s["chosen"].cpu().numpy().reshape(-1)
        kept = [i for i in range(chosen.size) if 0 <= chosen[i] < case["groups"]]
        kept.sort(key=lambda i: (chosen[i], i))
        order = torch.tensor(kept, dtype=torch.int64, device="cuda")
        rows = torch.zeros((chosen.size, case["d"]), device="cuda", dtype=f64)
        rows[: len(kept)] = s["x"].to(f64)[order // case["choices"]]
        return {"rows": rows, "slots": None, "order": None, "offsets": None}
    if op in ("back", "grad"):
        t, k, d = case["tokens"], case["choices"], case["d"]
        slots, weights = s["slots"].to(torch.int64), s["weights"].to(f64)
        total = torch.zeros((t, d), device="cuda", dtype=f64)
        rows = torch.zeros((t * k, d), device="cuda", dtype=f64)
        dots = torch.zeros((t, k), device="cuda", dtype=f64)
        for j in range(k):
            who = (slots[:, j] >= 0).nonzero()[:, 0]
            at = slots[who, j]
            if op == "back":
                total[who] += s["given_rows"][at].to(f64) * weights[who, j, None]
            else:
                given = s["given"][who].to(f64)
                rows[at] = given * weights[who, j, None]
                dots[who, j] = (given * s["given_rows"][at].to(f64)).sum(1)
                total[who] += s["given_sorted"][at].to(f64)
        return total if op == "back" else {"rows": rows, "weights": dots, "x": total}
    if case["x"] == "i8":
        q, scales = s["x"].to(f64), s["x_scales"].to(f64)
    else:
        x = s["x"].to(f64)
        most = x.abs().max(dim=1).values.clamp(min=1e-300)
        q, scales = (127 * x / most[:, None]).round(), most / 127
    x = q * scales[:, None]
    spans = [(0, case["m"])] if s["offsets"] is None else list(zip(s["offsets"].tolist()[:-1], s["offsets"].tolist()[1:]))
    y = torch.zeros((case["m"], case["n"]), device="cuda", dtype=f64)
    for e, (i, j) in enumerate(spans):
        if i < j:
            w = s["w"] if s["offsets"] is None else s["w"][e]
            scale = s["w_scales"] if s["offsets"] is None else s["w_scales"][e]
            y[i:j] = x[i:j] @ (w.to(f64) * scale.to(f64)[:, None]).t()
            if s["bias"] is not None:
                y[i:j] += (s["bias"] if s["offsets"] is None else s["bias"][e]).to(f64)
    return y
