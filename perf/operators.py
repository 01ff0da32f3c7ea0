"""Microscaled 4-bit operators of the expert FFN, as cases of one pass each.

An operand's elements are E2M1 values that share, in blocks of 32 along the reduction, a power of two:
with a = max |x| of the block, e = floor(log2 a) - 2 (within [-127, 127]), every element is x / 2^e rounded to the
nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code, larger ones to 6) times 2^e.

Kinds of case
  round_trip  quantise a tensor along its last or last but one axis, and the values it then stands for
  product     rows in bf16, quantised, times packed weights: one group, or ragged groups of rows with weights each
  gated       silu(x Wg) * (x Wu) * scale in one product over packed gate and up weights, activation in bf16
  experts     the whole expert FFN over packed weights; the activation stays in 4 bits between the products
  train       the FFN over bf16 weights that are quantised in the call, and the gradients of rows and weights: of the
              formula with the quantised operands in it, the quantisation itself passed straight through

Sizes are those of the repository's configurations (H=7168, H'=2048, top-8; hidden 2048, H'=768, 128 experts) and
generic ones between them.
"""
import random

import torch

own = False


def listed():
    return [
        # a decoding batch's rows before the gate and up projections: latency
        dict(name="round_trip_16x7168", kind="round_trip", G=1, rows=16, cols=7168, axis=-1, dtype="bf16"),
        # one projection of 32 experts, laid out [H, H'], with the reduction over H: what packing a model's weights costs
        dict(name="round_trip_32_experts", kind="round_trip", G=32, rows=7168, cols=2048, axis=-2, dtype="bf16"),
        # fp32 rows of odd length (a last block that is not full)
        dict(name="round_trip_odd_fp32", kind="round_trip", G=1, rows=1531, cols=1003, axis=-1, dtype="fp32"),
        # down projection of 16 decoded tokens, top-8 of 32 experts: a stream of the weights
        dict(name="product_decode", kind="product", G=32, rows=128, K=2048, N=7168, zipf=0.3, pad=1),
        # down projection of a prompt of 1531 tokens, ragged groups back to back
        dict(name="product_prefill", kind="product", G=32, rows=12248, K=2048, N=7168, zipf=0.5, pad=1),
        # one dense product, the largest: bound by the tensor cores
        dict(name="product_dense", kind="product", G=1, rows=8192, K=7168, N=4096, zipf=0.0, pad=1),
        # gate and up projections of the same decoding batch and of the same prompt (groups padded as the layer's are)
        dict(name="gated_decode", kind="gated", G=32, rows=128, K=7168, N=2048, zipf=0.3, pad=64),
        dict(name="gated_prefill", kind="gated", G=32, rows=12248, K=7168, N=2048, zipf=0.5, pad=128),
        # one token on the decoder's layer: the smallest call
        dict(name="experts_one_token", kind="experts", G=128, rows=8, K=2048, N=768, zipf=0.0, pad=1),
        # odd sizes everywhere
        dict(name="experts_odd", kind="experts", G=5, rows=333, K=1000, N=515, zipf=1.0, pad=1),
        # training step of the decoder's experts, padded groups
        dict(name="train_decoder", kind="train", G=128, rows=32768, K=2048, N=768, zipf=0.5, pad=128),
        # a dense block (shared expert) on an odd number of tokens
        dict(name="train_shared", kind="train", G=1, rows=777, K=1024, N=520, zipf=0.0, pad=1),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["round_trip", "product", "product", "gated", "gated", "experts", "experts", "train"])
    if kind == "round_trip":
        G = rng.choice([1, 1, _log_int(rng, 2, 32)])
        return dict(kind=kind, G=G, rows=_log_int(rng, 1, 7168), cols=_log_int(rng, 16, 4096 if G > 1 else 16384),
                    axis=rng.choice([-1, -2]), dtype=rng.choice(["bf16", "fp16", "fp32"]))
    if kind == "train":
        G = rng.choice([1, _log_int(rng, 2, 64)])
        return dict(kind=kind, G=G, rows=_log_int(rng, 64, 8192), K=128 * _log_int(rng, 2, 16), N=8 * _log_int(rng, 16, 128),
                    zipf=round(rng.uniform(0.0, 1.0), 2), pad=1 if G == 1 else rng.choice([64, 128]))
    G = rng.choice([1, _log_int(rng, 2, 32), _log_int(rng, 2, 32)])
    odd = rng.random() < 0.3
    step = 1 if odd else 64
    return dict(kind=kind, G=G, rows=_log_int(rng, 1, 8192), K=step * _log_int(rng, 256 // step, 7168 // step),
                N=step * _log_int(rng, 256 // step, 2048 // step), zipf=round(rng.uniform(0.0, 1.0), 2),
                pad=rng.choice([1, 64, 128]))


# ---- inputs -----------------------------------------------------------------------------------
DTYPES = dict(bf16=torch.bfloat16, fp16=torch.float16, fp32=torch.float32)


def _sizes(case):
    """Rows of the groups that hold tokens: `rows` in all, of a Zipf popularity."""
    p = [(i + 1.0) ** -case["zipf"] for i in range(case["G"])]
    total, sizes = sum(p), []
    for i in range(case["G"]):
        sizes.append(int(case["rows"] * sum(p[:i + 1]) / total + 0.5) - sum(sizes))
    return sizes


def _padded(n, pad):
    return (n + pad - 1) // pad * pad


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 1009 + 7)

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)

    if case["kind"] == "round_trip":
        shape = (case["rows"], case["cols"])
        x = normal(*(shape if case["G"] == 1 else (case["G"], *shape)), dtype=DTYPES[case["dtype"]])
        return dict(x=x)
    G, K, N, pad = case["G"], case["K"], case["N"], case["pad"]
    sizes = _sizes(case)
    random.Random(int(seed) * 31 + 5).shuffle(sizes)
    ends, at = [], 0
    live = torch.zeros(sum(_padded(n, pad) for n in sizes), 1, dtype=torch.bool)
    for n in sizes:
        live[at:at + n] = True
        at += _padded(n, pad)
        ends.append(at)
    live = live.cuda()
    d = dict(cu=torch.tensor(ends, dtype=torch.int32, device="cuda"), M=max(_padded(n, pad) for n in sizes),
             pads=torch.tensor([[e - _padded(n, pad) + n, _padded(n, pad) - n] for e, n in zip(ends, sizes)],
                               dtype=torch.int32, device="cuda"))
    # activations have channels that stand out; padding rows are zero
    channel = 1.0 + 9.0 * (torch.rand(K, device="cuda", generator=gen) < 0.01)
    d["x"] = (torch.randn(live.shape[0], K, device="cuda", generator=gen) * channel * live).bfloat16()
    if case["kind"] == "product":
        d["w"] = normal(G, N, K, scale=K ** -0.5)
        return d
    d["wg"], d["wu"] = normal(G, K, N, scale=K ** -0.5), normal(G, K, N, scale=K ** -0.5)
    d["scale"] = (0.05 + torch.rand(live.shape[0], device="cuda", generator=gen)) * live[:, 0]
    if case["kind"] != "gated":
        d["wd"] = normal(G, K, N, scale=N ** -0.5)
    if case["kind"] == "train":
        d["dy"] = (torch.randn(live.shape[0], K, device="cuda", generator=gen) * 0.01 * live).bfloat16()
    return d


# ---- plain form -------------------------------------------------------------------------------
def _quantised(x):
    """Values that x stands for once quantised along its last axis."""
    K = x.shape[-1]
    blocks = torch.nn.functional.pad(x.float(), (0, -K % 32)).unflatten(-1, (-1, 32))
    _, e = torch.frexp(blocks.abs().amax(-1, keepdim=True))            # a = m 2^e, m in [0.5, 1)
    e = (e - 3).clamp(-127, 127)
    y = torch.ldexp(blocks, -e).clamp(-6.0, 6.0)
    step = 0.5 * (1.0 + (y.abs() >= 2.0) + 2.0 * (y.abs() >= 4.0))
    return torch.ldexp(torch.round(y / step) * step, e).flatten(-2)[..., :K]


def _per_group(a, d, M):
    """Rows as [groups, M, columns], zeros behind each group's last; and where they came from."""
    rows = torch.arange(a.shape[0], device=a.device)
    g = torch.searchsorted(d["cu"].long(), rows, right=True)
    start = torch.cat([d["cu"].new_zeros(1), d["cu"][:-1]]).long()
    at = (g, rows - start[g])
    out = a.new_zeros(d["cu"].numel(), M, a.shape[1])
    out[at] = a
    return out, at


def _grouped(a, w, d):
    """a's rows of each group times that group's w [N, K], transposed."""
    rows, at = _per_group(a, d, d["M"])
    return torch.bmm(rows, w.transpose(1, 2))[at]


def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _act(x, wg, wu, d):
    gate, up = _grouped(x, wg, d), _grouped(x, wu, d)
    return _silu(gate) * up, gate, up


def _plain_train(s):
    x = _quantised(s["x"])
    wg, wu, wd = _quantised(s["wg"].transpose(1, 2)), _quantised(s["wu"].transpose(1, 2)), _quantised(s["wd"])
    act, gate, up = _act(x, wg, wu, s)
    act = _quantised(act.bfloat16())
    y = _grouped(act, wd, s)
    dy = s["dy"].float()
    dact = _grouped(dy, wd.transpose(1, 2), s)
    sig = 1.0 / (1.0 + torch.exp(-gate))
    dgate, dup = dact * up * sig * (1.0 + gate * (1.0 - sig)), dact * gate * sig
    dx = _grouped(dgate, wg.transpose(1, 2), s) + _grouped(dup, wu.transpose(1, 2), s)
    xt, dyt = _per_group(x, s, s["M"])[0].transpose(1, 2), _per_group(dy, s, s["M"])[0].transpose(1, 2)
    dwg, dwu = torch.bmm(xt, _per_group(dgate, s, s["M"])[0]), torch.bmm(xt, _per_group(dup, s, s["M"])[0])
    dwd = torch.bmm(dyt, _per_group(act, s, s["M"])[0])
    return tuple(t.bfloat16() for t in (y, dx, dwg, dwu, dwd))


# ---- the cases --------------------------------------------------------------------------------
def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    kind = case["kind"]
    if kind in ("round_trip", "train"):
        if kind == "train":
            for name in ("x", "wg", "wu", "wd"):
                s[name].requires_grad_(own)
        return s
    # weights, laid out once
    if own:
        from moonep_b200.ops import mx
        if kind == "product":
            s["w"] = mx.quantize(s["w"])
        else:
            s["wgu"] = mx.pack_gate_up(s.pop("wg"), s.pop("wu"))
            if kind == "experts":
                s["wd"] = mx.quantize(s["wd"])
    else:
        for name in {"w", "wd"} & s.keys():
            s[name] = _quantised(s[name])
        for name in {"wg", "wu"} & s.keys():
            s[name] = _quantised(s[name].transpose(1, 2))
    return s


def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if own:
        from moonep_b200.ops import mx
        if kind == "round_trip":
            return mx.quantize(s["x"], axis=case["axis"]).dequantize()
        if kind == "train":
            y = mx.expert_ffn(s["x"], s["wg"], s["wu"], s["wd"], s["cu"], pads=s["pads"])
            return (y.detach(), *torch.autograd.grad(y, (s["x"], s["wg"], s["wu"], s["wd"]), s["dy"]))
        x = mx.quantize(s["x"])
        if kind == "product":
            return mx.matmul(x, s["w"], s["cu"], pads=s["pads"])
        act, _, _ = mx.gateup_swiglu(x, s["wgu"], s["cu"], row_scale=s["scale"], quantize=kind == "experts", pads=s["pads"])
        return act if kind == "gated" else mx.matmul(act, s["wd"], s["cu"], pads=s["pads"])
    if kind == "round_trip":
        return _quantised(s["x"] if case["axis"] == -1 else s["x"].transpose(-1, -2)).bfloat16()
    if kind == "train":
        return _plain_train(s)
    x = _quantised(s["x"])
    if kind == "product":
        return _grouped(x, s["w"], s).bfloat16()
    act = (_act(x, s["wg"], s["wu"], s)[0] * s["scale"][:, None]).bfloat16()
    return act if kind == "gated" else _grouped(_quantised(act), s["wd"], s).bfloat16()


def work(case):
    size = 4 if case.get("dtype") == "fp32" else 2
    if case["kind"] == "round_trip":
        n = case["G"] * case["rows"] * case["cols"]
        return dict(bytes=n * (size + 2), flops=0)
    sizes = _sizes(case)
    used, rows, all_rows = sum(n > 0 for n in sizes), case["rows"], sum(_padded(n, case["pad"]) for n in sizes)
    KN, packed = case["K"] * case["N"], 17.0 / 32.0
    out = {"product": case["N"], "gated": case["N"]}.get(case["kind"], case["K"])
    products = {"product": 1, "gated": 2, "experts": 3, "train": 3}[case["kind"]]
    if case["kind"] == "train":       # x and dy read, y and dx written; weights read and their gradients written, all groups
        return dict(bytes=all_rows * case["K"] * 8 + case["G"] * KN * 12, flops=3 * products * 2 * rows * KN)
    return dict(bytes=all_rows * (case["K"] + out) * 2 + used * products * KN * packed, flops=products * 2 * rows * KN)


# ---- the definition in 64 bits ----------------------------------------------------------------
def _values64(x):
    """As _quantised, by comparing with the borders between neighbouring values."""
    K = x.shape[-1]
    full = torch.zeros(*x.shape[:-1], (K + 31) // 32 * 32, dtype=torch.float64, device=x.device)
    full[..., :K] = x
    b = full.view(*x.shape[:-1], -1, 32)
    a = b.abs().max(dim=-1, keepdim=True).values
    e = torch.floor(torch.log2(torch.where(a > 0, a, 1.0)))
    e = torch.where(torch.exp2(e) > a, e - 1, torch.where(torch.exp2(e + 1) <= a, e + 1, e)) - 2.0
    unit = torch.exp2(torch.where(a > 0, e, -127.0).clamp(min=-127.0))
    m = b.abs() / unit
    value = torch.zeros_like(m)
    for border, up, step in ((0.25, False, 0.5), (0.75, True, 0.5), (1.25, False, 0.5), (1.75, True, 0.5),
                             (2.5, False, 1.0), (3.5, True, 1.0), (5.0, False, 2.0)):
        value += step * ((m >= border) if up else (m > border))
    return (torch.sign(b) * value * unit).view(full.shape)[..., :K]


def exact(case, seed):
    d = _inputs(case, seed)
    kind = case["kind"]
    if kind == "round_trip":
        x = d["x"] if case["axis"] == -1 else d["x"].transpose(-1, -2).contiguous()
        if x.dim() == 3:
            return torch.stack([_values64(m) for m in x])
        return _values64(x)
    rows = d["x"].shape[0]
    ends = d["cu"].tolist()
    f64 = dict(dtype=torch.float64, device="cuda")
    width = case["K"] if kind in ("experts", "train") else case["N"]
    y = torch.zeros(rows, width, **f64)
    dx = torch.zeros(rows, case["K"], **f64) if kind == "train" else None
    grads = [torch.zeros(case["G"], case["K"], case["N"], **f64) for _ in range(3)] if kind == "train" else []
    for g, (a, b) in enumerate(zip([0] + ends[:-1], ends)):
        if a == b:
            continue
        x = _values64(d["x"][a:b])
        if kind == "product":
            y[a:b] = x @ _values64(d["w"][g]).T
            continue
        wg, wu = _values64(d["wg"][g].T.contiguous()), _values64(d["wu"][g].T.contiguous())
        gate, up = x @ wg.T, x @ wu.T
        act = gate * torch.sigmoid(gate) * up
        if kind != "train":
            act = act * d["scale"][a:b, None].double()
        if kind == "gated":
            y[a:b] = act
            continue
        act = _values64(act.bfloat16())          # the activation is rounded to bf16, then quantised
        wd = _values64(d["wd"][g])
        y[a:b] = act @ wd.T
        if kind == "train":
            dy = d["dy"][a:b].double()
            dact = dy @ wd
            sg = torch.sigmoid(gate)
            dgate, dup = dact * up * (sg + gate * sg * (1 - sg)), dact * gate * sg
            dx[a:b] = dgate @ wg + dup @ wu
            grads[0][g], grads[1][g], grads[2][g] = x.T @ dgate, x.T @ dup, dy.T @ act
    return (y, dx, *grads) if kind == "train" else y
