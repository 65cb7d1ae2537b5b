"""Cases of the routed products (tokens sorted by expert and back, 8-bit products by blocks of 128):
inputs, one pass through each operator in plain torch operations or through the library, the work
a pass cannot do without, and the results in 64 bits."""
import math
import sys
from pathlib import Path

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding step of 32 sequences: latency of the smallest sort; ids as topk gives them
        dict(name="route_step", op="route", tokens=32, top_k=8, experts=64, ids="i64", skew=0.0,
             drop=0.0),
        # a long batch over popular and rare experts, a twentieth of the pairs over capacity
        dict(name="route_prompt", op="route", tokens=65536, top_k=8, experts=256, ids="i32",
             skew=1.1, drop=0.05),
        # odd sizes in 32 bits, the weight applied before the expert
        dict(name="dispatch_odd", op="dispatch", tokens=1000, top_k=3, experts=16, width=1111,
             type="f32", weighted=True, skew=0.0, drop=0.1),
        # a training or prompt batch to its experts
        dict(name="dispatch_batch", op="dispatch", tokens=8192, top_k=8, experts=64, width=4096,
             type="bf16", weighted=False, skew=1.1, drop=0.0),
        # one decoding step back from its experts
        dict(name="combine_step", op="combine", tokens=32, top_k=8, experts=64, width=4096,
             type="f16", weighted=True, skew=0.0, drop=0.0),
        # the backward pass of a training batch: gradients of the experts' rows and of the weights
        dict(name="combine_grad_batch", op="combine_grad", tokens=8192, top_k=4, experts=64,
             width=4096, type="bf16", weighted=True, skew=1.1, drop=0.05),
        # a prompt batch to its experts in 8 bits
        dict(name="quantize_routed", op="quantize_routed", tokens=8192, top_k=8, experts=64,
             width=4096, type="bf16", skew=1.1, drop=0.0),
        # between the two products of an expert: silu(gate) * up in 8 bits, with unused rows behind
        dict(name="quantize_gated", op="quantize", rows=16384, spare=3000, width=2048, type="bf16",
             gated=True),
        # the experts' products of a prompt batch
        dict(name="product_prompt", op="product", tokens=4096, top_k=8, experts=64, n=2048, k=2048,
             type="bf16", skew=1.1, drop=0.0),
        # the experts' products of one decoding step: every chosen expert's weights for a few rows
        dict(name="product_step", op="product", tokens=16, top_k=8, experts=64, n=4096, k=2048,
             type="bf16", skew=0.0, drop=0.0),
        # a dense layer over a large batch
        dict(name="product_dense", op="product", tokens=8192, top_k=1, experts=1, n=8192, k=4096,
             type="bf16", skew=0.0, drop=0.0),
        # a dense layer for a single token
        dict(name="product_one", op="product", tokens=1, top_k=1, experts=1, n=4096, k=4096,
             type="f32", skew=0.0, drop=0.0),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["route", "dispatch", "combine", "combine_grad", "quantize_routed", "quantize",
                     "product", "product"])
    skew, drop = rng.choice([0.0, 0.6, 1.1]), rng.choice([0.0, 0.0, 0.05, 0.3])
    if op == "route":
        experts = log(8, 512)
        top_k = min(rng.randint(1, 16), experts)
        return dict(op=op, tokens=log(1, 524288 // top_k), top_k=top_k, experts=experts,
                    ids=rng.choice(["i32", "i64"]), skew=skew, drop=drop)
    if op == "quantize":
        width = log(32, 8192)
        rows = log(1, min(65536, (1 << 25) // width))
        return dict(op=op, rows=rows, spare=rng.choice([0, 1, rows // 4]), width=width,
                    type=rng.choice(["f32", "f16", "bf16"]), gated=rng.choice([False, True]))
    if op == "product":
        experts = rng.choice([1, log(2, 64)])
        top_k = min(rng.randint(1, 8), experts)
        n, k = log(64, 8192), log(64, 8192)
        while experts * n * k > 1 << 28:
            experts, top_k = (experts + 1) // 2, min(top_k, (experts + 1) // 2)
        most = max(1, min(16384, (1 << 37) // (n * k)) // top_k)
        return dict(op=op, tokens=log(1, most), top_k=top_k, experts=experts, n=n, k=k,
                    type=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    skew=rng.choice([0.0, 0.6]), drop=drop if experts > 1 else 0.0)
    experts = log(8, 256)
    top_k = min(rng.randint(1, 8), experts)
    width = log(64, 8192)
    types = ["f32", "f16", "bf16"] if op == "quantize_routed" else ["f64", "f32", "f16", "bf16"]
    case = dict(op=op, tokens=log(1, min(16384, (1 << 26) // (top_k * width))), top_k=top_k,
                experts=experts, width=width, type=rng.choice(types), skew=skew, drop=drop)
    if op != "quantize_routed":
        case["weighted"] = True if op == "combine_grad" else rng.choice([False, True])
    return case


# ----------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _ids(case, g):
    """Each token's top_k different experts (popularity ~ 1 / rank^skew in a random order), some
    of them dropped (-1)."""
    e, t = case["experts"], case["tokens"]
    rank = torch.randperm(e, generator=g, device="cuda") + 1
    noise = -torch.log(-torch.log(torch.rand(t, e, generator=g, device="cuda").clamp(1e-7, 1 - 1e-7)))
    ids = (noise - case["skew"] * torch.log(rank.float())).topk(case["top_k"], dim=1).indices
    if case["drop"]:
        off = torch.rand(ids.shape, generator=g, device="cuda") < case["drop"]
        ids = ids.masked_fill(off, -1)
    return ids.to(torch.int64 if case.get("ids") == "i64" else torch.int32).contiguous()


def _sort(ids, experts):
    """(expert_ptr, row_pair, pair_row) of the ids."""
    flat = ids.reshape(-1).long()
    kept = (flat >= 0) & (flat < experts)
    key = torch.where(kept, flat, torch.full_like(flat, experts))
    order = torch.sort(key, stable=True).indices
    ptr = torch.searchsorted(key[order], torch.arange(experts + 1, device=ids.device))
    rows = torch.arange(flat.numel(), device=ids.device)
    inside = rows < ptr[-1]
    row_pair = torch.where(inside, order, torch.full_like(order, -1))
    pair_row = torch.empty_like(order)
    pair_row[order] = torch.where(inside, rows, torch.full_like(rows, -1))
    return ptr.int(), row_pair.int(), pair_row.int()


def _values(g, rows, cols, dtype):
    """Rows of different sizes, as activations have them."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    return (x * torch.exp(torch.randn(rows, 1, generator=g, device="cuda"))).to(dtype)


def _blocks(k):
    return -(-k // BLOCK)


def _round_up(n, m):
    return -(-n // m) * m


def _in_blocks(x):
    """x [..., K] as [..., K / 128, 128], zeros behind the last column."""
    nb = _blocks(x.shape[-1])
    x = torch.nn.functional.pad(x, (0, nb * BLOCK - x.shape[-1]))
    return x.reshape(*x.shape[:-1], nb, BLOCK)


def _quantized(x):
    """(values in 8 bits, scales [K / 128, rows]) of x [rows, K] in 32 bits."""
    b = _in_blocks(x)
    tiny = torch.finfo(torch.float32).tiny
    # a quotient rounded once: dividing by a Python number would multiply by its reciprocal
    s = (b.abs().amax(-1) / torch.full((), E4M3_MAX, device=x.device)).clamp(min=tiny)
    q = (b / s[..., None]).reshape(x.shape[0], -1)[:, :x.shape[1]]
    return q.to(torch.float8_e4m3fn), s.t().contiguous()


def _eight_bits(rows, cols):
    """Storage of rows in 8 bits: a row begins every 16 bytes."""
    return torch.zeros(rows, _round_up(cols, 16), dtype=torch.float8_e4m3fn, device="cuda")


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    s = {"case": case, "op": op}
    if op == "quantize":
        rows = case["rows"] + case["spare"]
        s["x"] = _values(g, rows, case["width"] * (2 if case["gated"] else 1), TYPES[case["type"]])
        s["count"] = torch.tensor([case["rows"]], dtype=torch.int32, device="cuda")
        s["q"] = _eight_bits(rows, case["width"])
        s["scale"] = torch.zeros(_blocks(case["width"]), rows, device="cuda")
    else:
        ids = _ids(case, g)
        ptr, row_pair, pair_row = _sort(ids, case["experts"])
        pairs = case["tokens"] * case["top_k"]
        s["pairs"] = pairs
        if op == "route":
            s["ids"] = ids
            s["expert_ptr"] = torch.zeros_like(ptr)
            s["row_pair"] = torch.full_like(row_pair, -1)
            s["pair_row"] = torch.zeros_like(pair_row)
        elif op == "product":
            _prepare_product(s, case, g, ptr, pairs)
        else:
            s["expert_ptr"], s["pair_row"] = ptr, pair_row
            dtype = TYPES[case["type"]]
            acc = torch.float64 if dtype == torch.float64 else torch.float32
            w = torch.rand(case["tokens"], case["top_k"], generator=g, device="cuda", dtype=acc)
            if case.get("weighted"):
                s["w"] = (w / w.sum(1, keepdim=True)).contiguous()
            width, tokens = case["width"], case["tokens"]
            if op in ("dispatch", "quantize_routed", "combine_grad"):
                s["x"] = _values(g, tokens, width, dtype)
            if op in ("combine", "combine_grad"):
                s["h"] = _values(g, pairs, width, dtype)
            if op == "dispatch":
                s["y"] = torch.zeros(pairs, width, dtype=dtype, device="cuda")
            elif op == "combine":
                s["y"] = torch.zeros(tokens, width, dtype=dtype, device="cuda")
            elif op == "combine_grad":
                s["dh"] = torch.zeros(pairs, width, dtype=dtype, device="cuda")
                s["dw"] = torch.zeros(tokens, case["top_k"], dtype=acc, device="cuda")
            else:
                s["q"] = _eight_bits(pairs, width)
                s["scale"] = torch.zeros(_blocks(width), pairs, device="cuda")
    if own:
        s["call"] = _call(s)
    return s


def _prepare_product(s, case, g, ptr, rows):
    e, n, k = case["experts"], case["n"], case["k"]
    q, scale = _quantized(_values(g, rows, k, torch.float32))
    s["a"] = _eight_bits(rows, k)
    s["a"][:, :k] = q
    s["a_scale"] = scale
    # weights by blocks of 128 x 128, each expert's made by itself to keep the peak small
    s["b"] = torch.zeros(e, n, _round_up(k, 16), dtype=torch.float8_e4m3fn, device="cuda")
    s["b_scale"] = torch.empty(e, _blocks(n), _blocks(k), device="cuda")
    for i in range(e):
        w = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
        w = torch.nn.functional.pad(w, (0, _blocks(k) * BLOCK - k, 0, _blocks(n) * BLOCK - n))
        w = w.reshape(_blocks(n), BLOCK, _blocks(k), BLOCK)
        sw = w.abs().amax((1, 3)) / E4M3_MAX
        w = (w / sw[:, None, :, None]).reshape(_blocks(n) * BLOCK, -1)[:n, :k]
        s["b"][i, :, :k] = w.to(torch.float8_e4m3fn)
        s["b_scale"][i] = sw
    s["expert_ptr"] = ptr if e > 1 else None
    s["y"] = torch.zeros(rows, n, dtype=TYPES[case["type"]], device="cuda")
    # the most rows of one expert: the plain form computes the experts' products as one batch
    s["most"] = int((ptr[1:] - ptr[:-1]).max())


# --------------------------------------------------------------------------------------- the runs
def run(s):
    if own:
        s["call"].run(torch.cuda.current_stream().cuda_stream)
        return _outputs(s)
    return _PLAIN[s["op"]](s)


def _outputs(s):
    op, case = s["op"], s["case"]
    if op == "route":
        return s["expert_ptr"], s["row_pair"], s["pair_row"]
    if op in ("quantize", "quantize_routed"):
        return s["q"][:, :case["width"]], s["scale"]
    if op == "combine_grad":
        return s["dh"], s["dw"]
    return s["y"]


def _call(s):
    """The library's call for the state's operator, its arguments built once."""
    pkg = str(Path(__file__).resolve().parent.parent / "appt-spgemm-challenge_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from appt_spgemm import experts as ex

    op, case = s["op"], s["case"]
    if op == "quantize":
        return ex.Quantize(s["x"], s["q"][:, :case["width"]], s["scale"], rows_ptr=s["count"],
                           gate="silu" if case["gated"] else None)
    if op == "route":
        need = ex.route_workspace_bytes(case["tokens"], case["top_k"], case["experts"])
        s["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        return ex.Route(s["ids"], case["experts"], s["expert_ptr"], s["row_pair"], s["pair_row"],
                        s["workspace"])
    if op == "product":
        k = case["k"]
        return ex.ScaledProduct(s["a"][:, :k], s["a_scale"], s["b"][:, :, :k], s["b_scale"],
                                s["y"], expert_ptr=s["expert_ptr"])
    routes = ex.Routes(case["tokens"], case["top_k"], s["pair_row"])
    if op == "dispatch":
        return ex.Dispatch(routes, s["x"], s["y"], weights=s.get("w"))
    if op == "combine":
        return ex.Combine(routes, s["h"], s["y"], weights=s.get("w"))
    if op == "combine_grad":
        return ex.CombineGrad(routes, s["x"], s["h"], weights=s["w"], dh=s["dh"], dweights=s["dw"])
    return ex.DispatchQuantize(routes, s["x"], s["q"][:, :case["width"]], s["scale"])


# ------------------------------------------------------------------------------------- plain forms
def _plain_route(s):
    return _sort(s["ids"], s["case"]["experts"])


def _wide(x):
    return x if x.dtype == torch.float64 else x.float()


def _to_rows(s, value, like):
    """value [pairs, ...] at each kept pair's row; zeros where no pair is."""
    row = s["pair_row"].long()
    row = torch.where(row >= 0, row, torch.full_like(row, s["pairs"]))
    y = torch.zeros(s["pairs"] + 1, *value.shape[1:], dtype=like, device=value.device)
    y[row] = value.to(like)
    return y[:-1]


def _per_pair(s, x):
    return x.repeat_interleave(s["case"]["top_k"], dim=0)


def _from_rows(s, h):
    """h at each pair's row, zeros for dropped pairs."""
    row = s["pair_row"].long()
    return torch.where((row >= 0)[:, None], _wide(h)[row.clamp(min=0)], 0.0)


def _plain_dispatch(s):
    x = _per_pair(s, _wide(s["x"]))
    if "w" in s:
        x = x * s["w"].reshape(-1, 1)
    return _to_rows(s, x, s["y"].dtype)


def _plain_combine(s):
    h = _from_rows(s, s["h"])
    if "w" in s:
        h = h * s["w"].reshape(-1, 1)
    h = h.reshape(s["case"]["tokens"], s["case"]["top_k"], -1)
    return h.sum(1).to(s["y"].dtype)


def _plain_combine_grad(s):
    dy = _per_pair(s, _wide(s["x"]))
    dw = (dy * _from_rows(s, s["h"])).sum(1).reshape(s["dw"].shape)
    return _to_rows(s, dy * s["w"].reshape(-1, 1), s["dh"].dtype), dw


def _plain_quantize(s):
    x, width = _wide(s["x"]), s["case"]["width"]
    if s["case"]["gated"]:
        gate, up = x[:, :width], x[:, width:]
        x = gate / (1 + torch.exp(-gate)) * up
    q, scale = _quantized(x)
    inside = torch.arange(x.shape[0], device=x.device) < s["count"]
    q = torch.where(inside[:, None], q.float(), 0.0).to(torch.float8_e4m3fn)
    return q, torch.where(inside, scale, 0.0)


def _plain_quantize_routed(s):
    q, scale = _quantized(_wide(s["x"]))
    q = _to_rows(s, _per_pair(s, q.float()), torch.float32).to(torch.float8_e4m3fn)
    return q, _to_rows(s, _per_pair(s, scale.t()), torch.float32).t().contiguous()


def _plain_product(s):
    case = s["case"]
    n, k = case["n"], case["k"]
    a = _in_blocks(s["a"][:, :k].float()) * s["a_scale"].t()[:, :, None]
    a = a.reshape(a.shape[0], -1)[:, :k]
    b = s["b"][:, :, :k].float()
    sw = s["b_scale"].repeat_interleave(BLOCK, 1)[:, :n].repeat_interleave(BLOCK, 2)[:, :, :k]
    b = (b * sw).transpose(1, 2)
    if s["expert_ptr"] is None:
        return (a @ b[0]).to(s["y"].dtype)
    # rows padded to the same number for each expert, one batched product, and back
    ptr = s["expert_ptr"].long()
    r = torch.arange(a.shape[0], device=a.device)
    e = (torch.searchsorted(ptr, r, right=True) - 1).clamp(max=case["experts"] - 1)
    at = torch.where(r < ptr[-1], e * s["most"] + r - ptr[e], case["experts"] * s["most"])
    padded = torch.zeros(case["experts"] * s["most"] + 1, k, device=a.device)
    padded[at] = a
    y = torch.bmm(padded[:-1].reshape(case["experts"], -1, k), b).reshape(-1, n)
    y = torch.cat([y, torch.zeros(1, n, device=y.device)])[at]
    return torch.where((r < ptr[-1])[:, None], y, 0.0).to(s["y"].dtype)


_PLAIN = {"route": _plain_route, "dispatch": _plain_dispatch, "combine": _plain_combine,
          "combine_grad": _plain_combine_grad, "quantize": _plain_quantize,
          "quantize_routed": _plain_quantize_routed, "product": _plain_product}


# -------------------------------------------------------------------------------- work and 64 bits
def work(case):
    op = case["op"]
    if op == "quantize":
        size = TYPES[case["type"]].itemsize
        rows, width = case["rows"], case["width"]
        values = rows * width
        return {"bytes": values * (size * (2 if case["gated"] else 1) + 1)
                + 4 * rows * _blocks(width), "flops": values * (8 if case["gated"] else 3)}
    t, k, e = case["tokens"], case["top_k"], case["experts"]
    pairs = t * k
    kept = pairs * (1 - case["drop"])
    if op == "route":
        return {"bytes": pairs * (8 if case["ids"] == "i64" else 4) + 4 * pairs + 4 * kept
                + 4 * (e + 1), "flops": pairs}
    if op == "product":
        n, kk = case["n"], case["k"]
        # experts with a row at all, if they are equally popular
        used = e * (1 - (1 - k * (1 - case["drop"]) / e) ** t) if e > 1 else 1
        out = TYPES[case["type"]].itemsize
        return {"bytes": kept * (kk + 4 * _blocks(kk) + n * out)
                + used * (n * kk + 4 * _blocks(n) * _blocks(kk)), "flops": 2 * kept * n * kk}
    size, width = TYPES[case["type"]].itemsize, case["width"]
    acc = 8 if case["type"] == "f64" else 4
    index = pairs * (4 + (acc if case.get("weighted") else 0))
    if op == "quantize_routed":
        return {"bytes": t * width * size + kept * (width + 4 * _blocks(width)) + index,
                "flops": 3 * t * width}
    moved = (t + kept) * width * size
    if op == "combine_grad":
        return {"bytes": moved + kept * width * size + index + acc * pairs,
                "flops": 3 * kept * width}
    return {"bytes": moved + index, "flops": kept * width * (2 if case.get("weighted") else 1)}


def _e4m3(v):
    """v in 64 bits at the nearest value of e4m3 (ties to even), still in 64 bits."""
    exponent = torch.frexp(v.abs().clamp(min=2.0 ** -6)).exponent
    step = torch.ldexp(torch.ones_like(v), exponent - 4)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_quantized(x):
    rows, width = x.shape
    nb = _blocks(width)
    b = torch.zeros(rows, nb * BLOCK, dtype=torch.float64, device=x.device)
    b[:, :width] = x
    b = b.view(rows, nb, BLOCK)
    top = b.abs().max(-1).values
    scale = (top / E4M3_MAX).float().double()  # a scale is held in 32 bits
    q = _e4m3(torch.where(top[..., None] > 0, b / scale[..., None], 0.0))
    return q.view(rows, -1)[:, :width], scale


def exact(case, seed):
    op = case["op"]
    if op == "route":
        return None
    s = prepare(case, seed)
    if op == "quantize":
        x, width, rows = s["x"].double(), case["width"], case["rows"]
        if case["gated"]:
            x = x[:, :width] * torch.sigmoid(x[:, :width]) * x[:, width:]
        q, scale = _exact_quantized(x)
        q[rows:], scale[rows:] = 0, 0
        return q, scale.t()
    if op == "product":
        return _exact_product(case, s)
    # the routing as a sparse matrix: (row of the sorted order, token) of each kept pair
    pair = torch.nonzero(s["pair_row"] >= 0).flatten()
    row, token = s["pair_row"][pair].long(), pair // case["top_k"]
    w = s["w"].double().flatten()[pair] if "w" in s else torch.ones_like(pair).double()
    if op == "combine":
        y = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
        return y.index_add_(0, token, s["h"].double()[row] * w[:, None])
    x = s["x"].double()
    y = torch.zeros(s["pairs"], case["width"], dtype=torch.float64, device="cuda")
    if op == "quantize_routed":
        q, scale = _exact_quantized(x)
        ys = torch.zeros(s["pairs"], scale.shape[1], dtype=torch.float64, device="cuda")
        y[row], ys[row] = q[token], scale[token]
        return y, ys.t()
    y[row] = x[token] * w[:, None]
    if op == "dispatch":
        return y
    dw = torch.zeros(s["pairs"], dtype=torch.float64, device="cuda")
    dw[pair] = torch.einsum("pc,pc->p", x[token], s["h"].double()[row])
    return y, dw.view(case["tokens"], case["top_k"])


def _exact_product(case, s):
    n, k = case["n"], case["k"]
    y = torch.zeros(s["pairs"], n, dtype=torch.float64, device="cuda")
    ptr = [0, s["pairs"]] if s["expert_ptr"] is None else s["expert_ptr"].tolist()
    column = torch.arange(k, device="cuda") // BLOCK
    line = torch.arange(n, device="cuda") // BLOCK
    a = s["a"][:, :k].double() * s["a_scale"].double()[column].t()
    for e in range(case["experts"]):
        if ptr[e + 1] > ptr[e]:
            b = s["b"][e, :, :k].double() * s["b_scale"][e].double()[line][:, column]
            y[ptr[e]:ptr[e + 1]] = a[ptr[e]:ptr[e + 1]] @ b.t()
    return y
