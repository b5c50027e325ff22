"""The training-step operators' cases: what is measured of them, and their plain forms.

Five operators: the norm of a list of gradients with its clipping factor, an
AdamW step over a list of tensors with its states in 32 bits, the same step
with its states in 8 bits, the norms after and before a block fused with the
block's gate and residual scale, and that operator's gradients.

``run`` computes the plain form (elementary torch operations, in 32 bits or
more) where ``own`` is false, and calls the package's operators where it is
true.  ``exact`` restates each operator in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}

# AdamW's constants in every case.
BETA1, BETA2, EPS, DECAY, LR = 0.9, 0.95, 1e-8, 0.1, 3e-4

# 8-bit states: values a block, and the code value that stands for a block's largest.
BLOCK, TOP = 256, 256.0


# ---------------------------------------------------------------------------
# the cases


def listed():
    return [
        # the global norm of a small fine-tuned part: a few odd tensors, packed
        # one behind the other, where latency counts
        {"name": "norm few odd f32", "op": "grad_norm", "sizes": "7,4097,1,12800,333",
         "grad": "f32", "packed": True},
        # the global norm of a whole model's gradients: 32 layers of width 1024
        {"name": "norm model bf16", "op": "grad_norm", "layers": 32, "width": 1024, "vocab": 8192,
         "grad": "bf16", "packed": False},
        # the step of a small fine-tuned part: bias and norm vectors of odd sizes
        {"name": "adamw few odd f32", "op": "adamw", "sizes": "1025,64,4096,1,777,10000",
         "param": "f32", "grad": "f32", "master": False, "packed": True, "step": 0},
        # the step of a narrow model in mixed precision: many tensors of middling size
        {"name": "adamw narrow bf16+master", "op": "adamw", "layers": 16, "width": 256,
         "vocab": 4096, "param": "bf16", "grad": "bf16", "master": True, "packed": False,
         "step": 100},
        # the step of a whole model in 32 bits
        {"name": "adamw model f32", "op": "adamw", "layers": 8, "width": 1024, "vocab": 8192,
         "param": "f32", "grad": "f32", "master": False, "packed": False, "step": 1000},
        # 8-bit states on odd tensors that end inside a block
        {"name": "adamw8 few odd f32", "op": "adamw8", "sizes": "257,1000,31,65537,5",
         "param": "f32", "grad": "f32", "master": False, "packed": True, "step": 3},
        # 8-bit states for a whole model whose parameters are bf16
        {"name": "adamw8 model bf16", "op": "adamw8", "layers": 8, "width": 1024, "vocab": 8192,
         "param": "bf16", "grad": "bf16", "master": False, "packed": False, "step": 1000},
        # one new token of a served model: both norms, weights only
        {"name": "block one token bf16", "op": "block", "rows": 1, "width": 4096, "x": "bf16",
         "h": "bf16", "gate": "none", "strided": False},
        # a training batch: the branch and its gate are the halves of one projection
        {"name": "block batch bf16 token gate", "op": "block", "rows": 8192, "width": 4096,
         "x": "bf16", "h": "bf16", "gate": "token", "strided": True},
        # an odd width, a 32-bit residual stream, one gate row a sequence of the batch
        {"name": "block odd f32/bf16 batch gate", "op": "block", "rows": 1533, "width": 1023,
         "x": "f32", "h": "bf16", "gate": "batch3", "strided": False},
        # gradients of the training batch
        {"name": "block grad batch bf16", "op": "block_grad", "rows": 8192, "width": 4096,
         "x": "bf16", "h": "bf16", "gate": "token", "strided": True},
        # gradients of a small odd batch whose one gate row serves every token
        {"name": "block grad odd f16 channel gate", "op": "block_grad", "rows": 777, "width": 1535,
         "x": "f16", "h": "f16", "gate": "channel", "strided": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["grad_norm", "adamw", "adamw8", "block", "block_grad"])
    if op in ("block", "block_grad"):
        width = _log(rng, 48, 8192)
        if rng.random() < 0.6:
            width = max(8, width // 8 * 8)
        rows = _log(rng, 1, min(16384, (1 << 25) // width))
        x, h = rng.choice([("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"),
                           ("f32", "f16")])
        gate = rng.choice(["none", "token", "channel", "batch"])
        if gate == "batch":
            groups = rng.choice([2, 3, 5, 16])
            rows = max(1, rows // groups) * groups
            gate = "batch%d" % groups
        return {"op": op, "rows": rows, "width": width, "x": x, "h": h, "gate": gate,
                "strided": rng.random() < 0.3}
    c = {"op": op, "packed": rng.random() < 0.4}
    if rng.random() < 0.5:
        c["sizes"] = ",".join(str(_log(rng, 1, 300000)) for _ in range(rng.randint(1, 24)))
    else:
        c["width"] = rng.choice([64, 96, 128, 200, 256, 384, 512, 640])
        c["layers"] = rng.randint(1, 8)
        c["vocab"] = rng.choice([1000, 4096, 8192])
    c["grad"] = rng.choice(["f32", "bf16", "f16"])
    if op != "grad_norm":
        c["param"] = rng.choice(["f32", "bf16", "f16"])
        c["master"] = c["param"] != "f32" and rng.random() < 0.6
        c["step"] = rng.choice([0, 1, 17, 1000, 50000])
    return c


def _sizes(case):
    """The elements of each tensor of a list: those named, or a decoder's
    (an embedding, then six matrices and two norm vectors a layer)."""
    if "sizes" in case:
        return [int(s) for s in case["sizes"].split(",")]
    d = case["width"]
    return [case["vocab"] * d] + ([d * d] * 4 + [4 * d * d] * 2 + [d] * 2) * case["layers"]


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    op = case["op"]
    if op in ("block", "block_grad"):
        r, d, bx, bh = case["rows"], case["width"], BYTES[case["x"]], BYTES[case["h"]]
        g = _gate_rows(case)
        if op == "block":
            # x, h, gate and the two weights; y, z and the two statistics
            nbytes = r * d * (bx + bh + bx + bh) + g * d * bh + 2 * d * bh + 8 * r
            flops = 12 * r * d
        else:
            # y, h, gate, weights, dy, dz, statistics; dx, dh, dgate and the weights' gradients
            nbytes = r * d * (3 * bx + 3 * bh) + 2 * g * d * bh + 4 * d * bh + 8 * r
            flops = 30 * r * d
        return {"bytes": nbytes, "flops": flops}
    sizes = _sizes(case)
    n = sum(sizes)
    if op == "grad_norm":
        return {"bytes": n * BYTES[case["grad"]] + 8, "flops": 2 * n}
    per = 2 * BYTES[case["param"]] + BYTES[case["grad"]]
    if case["master"]:  # the parameter's copy is only written
        per = BYTES[case["param"]] + 8 + BYTES[case["grad"]]
    if op == "adamw":
        return {"bytes": n * (per + 16) + 24, "flops": 14 * n}
    return {"bytes": n * (per + 4) + 16 * sum(_blocks(k) for k in sizes) + 24, "flops": 40 * n}


# ---------------------------------------------------------------------------
# the inputs


def _rng(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _list(sizes, dtype, packed, fill):
    """Tensors of these sizes as views of one buffer: each at a boundary of 256
    elements, or packed one behind the other as in a flattened shard."""
    step = 1 if packed else 256
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // step) * step
    flat = torch.zeros(at, dtype=dtype, device="cuda")
    views = [flat[s:s + n] for s, n in zip(starts, sizes)]
    for v in views:
        v.copy_(fill(v.numel()))
    return flat, views


def prepare(case, seed):
    g = _rng(seed)
    randn = lambda *n: torch.randn(*n, device="cuda", generator=g)  # noqa: E731
    rand = lambda *n: torch.rand(*n, device="cuda", generator=g)  # noqa: E731
    s = {"case": dict(case), "op": case["op"]}
    if case["op"] in ("block", "block_grad"):
        return _prepare_block(case, s, randn)
    sizes, packed = _sizes(case), case["packed"]
    grad = DTYPES[case["grad"]]
    # a tensor's gradients have a scale of their own, between 1e-4 and 1e-2
    s["grads_flat"], s["grads"] = _list(sizes, grad, packed,
                                        lambda n: randn(n) * 10.0 ** (-4 + 2 * rand(1)))
    if case["op"] == "grad_norm":
        s["max_norm"] = 1.0
        return s
    param = DTYPES[case["param"]]
    s["params_flat"], s["params"] = _list(sizes, param, packed, lambda n: 0.02 * randn(n))
    s["master_flat"], s["master"] = None, None
    if case["master"]:
        s["master_flat"] = s["params_flat"].float()
        s["master_flat"] += 1e-5 * randn(s["master_flat"].numel()) * (s["master_flat"] != 0)
        base = s["params_flat"].data_ptr()
        at = [(p.data_ptr() - base) // p.element_size() for p in s["params"]]
        s["master"] = [s["master_flat"][a:a + n] for a, n in zip(at, sizes)]
    first = case["step"] == 0
    if case["op"] == "adamw":
        s["m_flat"], s["m"] = _list(sizes, torch.float32, packed,
                                    lambda n: 1e-3 * randn(n) * (not first))
        s["v_flat"], s["v"] = _list(sizes, torch.float32, packed,
                                    lambda n: 1e-5 * randn(n).square() * (not first))
    else:
        s["m_flat"], s["m"] = _list(sizes, torch.float8_e4m3fn, packed,
                                    lambda n: (60 * randn(n)).clamp(-TOP, TOP) * (not first))
        s["v_flat"], s["v"] = _list(sizes, torch.float8_e4m3fn, packed,
                                    lambda n: (30 * randn(n).square()).clamp(0.002, TOP)
                                    * (not first))
        s["m_top_flat"], s["m_top"] = _list([_blocks(n) for n in sizes], torch.float32, packed,
                                            lambda n: 4e-3 * (0.5 + rand(n)) * (not first))
        s["v_top_flat"], s["v_top"] = _list([_blocks(n) for n in sizes], torch.float32, packed,
                                            lambda n: 1e-4 * (0.5 + rand(n)) * (not first))
        s["seed"] = (int(seed) * 0x9E3779B97F4A7C15 + 12345) & 0x7FFFFFFFFFFFFFFF
    s["step"] = torch.tensor([case["step"]], dtype=torch.int64, device="cuda")
    s["lr"] = torch.tensor([LR], dtype=torch.float32, device="cuda")
    s["scale"] = 0.25 + 0.5 * rand(1)  # the clipping factor that the norm left on the device
    # vectors (norms, biases) are not decayed
    s["decay"] = [DECAY if n > case.get("width", 1024) else 0.0 for n in sizes]
    return s


def _gate_rows(case):
    gate = case["gate"]
    return {"none": 0, "token": case["rows"], "channel": 1}.get(gate) if not gate.startswith(
        "batch") else int(gate[5:])


def _prepare_block(case, s, randn):
    r, d, tx, th = case["rows"], case["width"], DTYPES[case["x"]], DTYPES[case["h"]]
    groups = _gate_rows(case)
    s["x"] = randn(r, d).to(tx)
    if case["strided"]:  # the halves of one projection's output
        both = randn(r, 2 * d).to(th)
        s["h"], gate = both[:, :d], both[:, d:]
    else:
        s["h"], gate = randn(r, d).to(th), None
    s["gate"] = None
    if groups == r and gate is not None:
        s["gate"] = gate
    elif groups:
        s["gate"] = randn(groups, d).to(th)
    s["post_weight"] = (1 + 0.1 * randn(d)).to(th)
    s["pre_weight"] = (1 + 0.1 * randn(d)).to(th)
    s["eps"], s["residual_scale"], s["branch_scale"] = 1e-6, 1.0, 0.5
    if case["op"] == "block_grad":
        # what the forward pass left: y and the two rows' statistics
        h = s["h"].float()
        s["post_rstd"] = (h.square().mean(1) + s["eps"]).rsqrt()
        u = h * s["post_rstd"][:, None] * s["post_weight"].float()
        y = s["x"].float() * s["residual_scale"] + s["branch_scale"] * _spread(s["gate"], r) * u
        s["pre_rstd"] = (y.square().mean(1) + s["eps"]).rsqrt()
        s["y"] = y.to(tx)
        del s["x"], u, y, h
        s["dy"] = (0.1 * randn(r, d)).to(tx)
        s["dz"] = (0.1 * randn(r, d)).to(th)
    return s


def _spread(gate, rows):
    """The gate for every row in 32 bits: each of its rows serves a run of rows."""
    if gate is None:
        return 1.0
    g = gate.float()
    return g.repeat_interleave(rows // g.shape[0], 0) if g.shape[0] != rows else g


# ---------------------------------------------------------------------------
# one pass


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    if "call" not in s:  # the handle that a program keeps for its buffers
        s["call"], s["result"] = _bind(s)
    s["call"]()
    return s["result"]


def _bind(s):
    from loom_b200.build import load_train
    ops, op = load_train(), s["op"]
    stream = torch.cuda.current_stream()
    if op == "grad_norm":
        call, out = ops["grad_norm"].bind(grads=s["grads"], max_norm=s["max_norm"], stream=stream)
        return call, {"norm": out}
    if op == "adamw":
        call, _ = ops["adamw"].bind(
            params=s["params"], grads=s["grads"], exp_avg=s["m"], exp_avg_sq=s["v"],
            master=s["master"], step=s["step"], lr=s["lr"], betas=(BETA1, BETA2), eps=EPS,
            weight_decay=s["decay"], grad_scale=s["scale"], stream=stream)
        return call, _updated(s)
    if op == "adamw8":
        call, _ = ops["adamw8"].bind(
            params=s["params"], grads=s["grads"], exp_avg=s["m"], exp_avg_sq=s["v"],
            exp_avg_top=s["m_top"], exp_avg_sq_top=s["v_top"], master=s["master"], step=s["step"],
            lr=s["lr"], betas=(BETA1, BETA2), eps=EPS, weight_decay=s["decay"],
            grad_scale=s["scale"], seed=s["seed"], stream=stream)
        return call, _updated(s)
    if op == "block":
        call, out = ops["block_norm"].bind(
            x=s["x"], h=s["h"], gate=s["gate"], post_weight=s["post_weight"],
            pre_weight=s["pre_weight"], eps=s["eps"], residual_scale=s["residual_scale"],
            branch_scale=s["branch_scale"], stream=stream)
        return call, {"y": out.y, "z": out.z, "post_rstd": out.post_rstd,
                      "pre_rstd": out.pre_rstd}
    call, out = ops["block_norm_backward"].bind(
        y=s["y"], h=s["h"], gate=s["gate"], post_weight=s["post_weight"],
        pre_weight=s["pre_weight"], post_rstd=s["post_rstd"], pre_rstd=s["pre_rstd"], dy=s["dy"],
        dz=s["dz"], residual_scale=s["residual_scale"], branch_scale=s["branch_scale"],
        stream=stream)
    return call, {"dx": out.dx, "dh": out.dh, "dgate": out.dgate,
                  "dpost_weight": out.dpost_weight, "dpre_weight": out.dpre_weight}


def _updated(s):
    """What a step leaves: the state's own buffers."""
    names = ["params_flat", "m_flat", "v_flat", "step"]
    names += ["master_flat"] if s["master"] is not None else []
    names += ["m_top_flat", "v_top_flat"] if s["op"] == "adamw8" else []
    return {k.replace("_flat", ""): s[k] for k in names}


def _plain(s):
    if s["op"] == "grad_norm":
        return _plain_norm(s)
    if s["op"] in ("adamw", "adamw8"):
        return _plain_adamw(s)
    return _plain_block(s) if s["op"] == "block" else _plain_block_grad(s)


def _plain_norm(s):
    g = torch.cat([t.float() for t in s["grads"]])
    norm = (g * g).sum(dtype=torch.float64).sqrt()
    scale = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm))
    return {"norm": torch.stack([norm, scale]).float()}


def _plain_adamw(s):
    sizes = [t.numel() for t in s["params"]]
    eight = s["op"] == "adamw8"
    old = s["master"] if s["master"] is not None else s["params"]
    p = torch.cat([t.float() for t in old])
    g = torch.cat([t.float() for t in s["grads"]]) * s["scale"]
    if eight:
        m, v = _opened(s["m"], s["m_top"]), _opened(s["v"], s["v_top"])
    else:
        m, v = torch.cat(s["m"]), torch.cat(s["v"])
    s["step"] += 1
    t = s["step"].double()
    lr = s["lr"].double()
    a = (lr / (1 - BETA1 ** t)).float()
    c = (1 / (1 - BETA2 ** t).sqrt()).float()
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    keep = torch.cat([(1 - lr * w).float().expand(n) for w, n in zip(s["decay"], sizes)])
    p = p * keep - a * (m / (v.sqrt() * c + EPS))
    if eight:
        key = _key(s["seed"], s["step"])
        rnd = torch.split(_random(key, sizes), [_blocks(n) for n in sizes])
        _close(m, sizes, s["m"], s["m_top"], rnd, 0)
        _close(v, sizes, s["v"], s["v_top"], rnd, 16)
    else:
        _put(m, s["m"])
        _put(v, s["v"])
    _put(p, s["params"])
    if s["master"] is not None:
        _put(p, s["master"])
    return _updated(s)


def _put(flat, tensors):
    """The values of a list, rounded to its tensors' type."""
    torch._foreach_copy_(tensors, list(torch.split(flat, [t.numel() for t in tensors])))


def _padded(t):
    """A tensor's values in 32 bits as rows of one block."""
    n = t.numel()
    return torch.nn.functional.pad(t.float(), (0, _blocks(n) * BLOCK - n)).view(-1, BLOCK)


def _opened(codes, tops):
    """8-bit states as values: code times the block's largest over TOP."""
    return torch.cat([(_padded(c) * (t * (1 / TOP))[:, None]).view(-1)[:c.numel()]
                      for c, t in zip(codes, tops)])


def _close(flat, sizes, codes, tops, rnd, shift):
    [_close_one(x, c, t, r, shift)
     for x, c, t, r in zip(torch.split(flat, sizes), codes, tops, rnd)]


def _close_one(x, codes, tops, rnd, shift):
    """Values to codes, each rounded up or down by its 16 random bits."""
    x = _padded(x)
    top = x.abs().amax(1)
    top = torch.where(top < 2.0 ** -100, 0.0, top)
    inv = torch.where(top > 0, torch.reciprocal(top) * TOP, 0.0)
    a = x.abs() * inv[:, None]
    low = a < 2.0 ** -6  # below the smallest normal code: one spacing down to zero
    bits = (a + torch.where(low, 2.0 ** -6, 0.0)).view(torch.int32).long()
    r = (((rnd >> shift) & 0xFFFF) << 4) + 8
    code = ((bits + r) >> 20) - (120 << 3) - torch.where(low, 8, 0)
    if shift:  # a second moment above zero stays above it
        code = torch.maximum(code, (x > 0).long())
    code = code + torch.where(x < 0, 128, 0)
    n = codes.numel()
    codes.copy_(code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1)[:n])
    tops.copy_(top)


U32 = 0xFFFFFFFF


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & U32
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & U32
    return x ^ (x >> 16)


def _key(seed, step):
    """The step's 32-bit key from the 64-bit seed and the step's number."""
    k = _mix(torch.full_like(step, (seed & U32) ^ 0x9E3779B9))
    k = _mix(k ^ (seed >> 32))
    k = _mix(k ^ (step & U32))
    return _mix(k ^ (step >> 32))


def _random(key, sizes):
    """32 random bits a value, as rows of one block: the blocks are counted
    through the list; eight neighbours share one full mix."""
    count = torch.arange(sum(_blocks(n) for n in sizes) * 32, device="cuda")
    h = _mix((_mix(count) + key) & U32)
    x = (h[:, None] + torch.arange(8, device="cuda") * 0x9E3779B9) & U32
    x = x ^ (x >> 17)
    x = (x * 0xBB67AE85) & U32
    return (x ^ (x >> 15)).view(-1, BLOCK)


def _plain_block(s):
    rows, tx, th = s["x"].shape[0], s["x"].dtype, s["h"].dtype
    h = s["h"].float()
    post_rstd = 1 / (h.square().mean(1) + s["eps"]).sqrt()
    u = h * post_rstd[:, None] * s["post_weight"].float()
    y = s["residual_scale"] * s["x"].float() + s["branch_scale"] * (_spread(s["gate"], rows) * u)
    pre_rstd = 1 / (y.square().mean(1) + s["eps"]).sqrt()
    z = y * pre_rstd[:, None] * s["pre_weight"].float()
    return {"y": y.to(tx), "z": z.to(th), "post_rstd": post_rstd, "pre_rstd": pre_rstd}


def _plain_block_grad(s):
    rows, tx, th = s["y"].shape[0], s["y"].dtype, s["h"].dtype
    y, h, dz = s["y"].float(), s["h"].float(), s["dz"].float()
    w_post, w_pre = s["post_weight"].float(), s["pre_weight"].float()
    r_post, r_pre = s["post_rstd"][:, None], s["pre_rstd"][:, None]
    gate, scale = _spread(s["gate"], rows), s["branch_scale"]
    n = y * r_pre
    t = dz * w_pre
    d = s["dy"].float() + r_pre * (t - n * (t * n).mean(1, keepdim=True))
    k = h * r_post
    t = scale * (gate * d) * w_post
    dh = r_post * (t - k * (t * k).mean(1, keepdim=True))
    dgate = None
    if s["gate"] is not None:
        dgate = scale * d * (k * w_post)
        groups = s["gate"].shape[0]
        if groups != rows:
            dgate = dgate.view(groups, rows // groups, -1).sum(1, dtype=torch.float64)
        dgate = dgate.to(th)
    return {"dx": (s["residual_scale"] * d).to(tx), "dh": dh.to(th), "dgate": dgate,
            "dpost_weight": (scale * gate * d * k).sum(0, dtype=torch.float64).to(th),
            "dpre_weight": (dz * n).sum(0, dtype=torch.float64).to(th)}


# ---------------------------------------------------------------------------
# 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "grad_norm":
        total = sum(float(torch.dot(g.double(), g.double())) for g in s["grads"])
        norm = math.sqrt(total)
        pair = [norm, min(1.0, s["max_norm"] / norm)]
        return {"norm": torch.tensor(pair, dtype=torch.float64)}
    if case["op"] in ("adamw", "adamw8"):
        return _exact_adamw(s, case["op"] == "adamw8")
    if case["op"] == "block":
        return _exact_block(s)
    return _exact_block_grad(s)


def _exact_adamw(s, eight):
    """One step from what prepare() made, tensor by tensor.  A code's value
    hangs on a border and its random bits; the 64-bit step gives it by the
    grid's own spacing."""
    t = int(s["step"]) + 1
    lr, scale = float(s["lr"]), float(s["scale"])
    flat = {k: s[k].double() for k in ("params_flat", "m_flat", "v_flat")}
    if s["master"] is not None:
        flat["master_flat"] = s["master_flat"].double()
    if eight:
        flat |= {k: s[k].double() for k in ("m_top_flat", "v_top_flat")}
    at = lambda view, base: view.storage_offset() - base.storage_offset()  # noqa: E731
    block0 = 0
    for i, p in enumerate(s["params"]):
        n, o = p.numel(), at(p, s["params_flat"])
        old = (s["master"][i] if s["master"] is not None else p).double()
        g = s["grads"][i].double() * scale
        m, v = s["m"][i].double(), s["v"][i].double()
        if eight:
            owner = torch.arange(n, device="cuda") // BLOCK
            m = m * s["m_top"][i].double()[owner] / TOP
            v = v * s["v_top"][i].double()[owner] / TOP
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g * g
        step = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
        new = old - lr * s["decay"][i] * old - lr * step
        flat["params_flat"][o:o + n] = new
        if s["master"] is not None:
            flat["master_flat"][o:o + n] = new
        if eight:
            b = at(s["m_top"][i], s["m_top_flat"])
            bits = _exact_bits(s["seed"], t, block0, n)
            for x, name, half in ((m, "m", bits % 65536), (v, "v", bits // 65536)):
                top = torch.zeros(_blocks(n), dtype=torch.float64, device="cuda")
                top.scatter_reduce_(0, owner, x.abs(), "amax")
                flat[name + "_top_flat"][b:b + _blocks(n)] = top
                flat[name + "_flat"][o:o + n] = _exact_code(x, top[owner], half, name == "v")
            block0 += _blocks(n)
        else:
            flat["m_flat"][o:o + n], flat["v_flat"][o:o + n] = m, v
    out = {k.replace("_flat", ""): x for k, x in flat.items()}
    out["step"] = None
    return out


def _exact_code(x, top, half, second):
    a = torch.where(top >= 2.0 ** -100, x.abs() * TOP / top.clamp_min(2.0 ** -100), 0.0)
    unit = torch.pow(2.0, torch.frexp(a)[1].double().clamp_min(-5) - 4)
    down = torch.floor(a / unit)
    up = (a / unit - down) * 2 ** 20 + half * 16 + 8 >= 2 ** 20
    q = (down + up) * unit
    if second:
        q = torch.where((q == 0) & (x > 0), 2.0 ** -9, q)
    return torch.copysign(q, x)


def _exact_bits(seed, step, block0, n):
    """The random words of one tensor's values, from the generator's definition."""
    def full(x):
        for mul, shift in ((0x6A09E667, 16), (0xBB67AE85, 15)):
            x = (torch.bitwise_xor(x, x // 2 ** shift) * mul) % 2 ** 32
        return torch.bitwise_xor(x, x // 2 ** 16)

    key = torch.tensor(0x9E3779B9 ^ (seed % 2 ** 32), device="cuda")
    for word in (seed // 2 ** 32, step % 2 ** 32, step // 2 ** 32):
        key = torch.bitwise_xor(full(key), torch.tensor(word, device="cuda"))
    key = full(key)
    i = torch.arange(n, device="cuda")
    h = full((full(block0 * 32 + i // 8) + key) % 2 ** 32)
    x = (h + (i % 8) * 0x9E3779B9) % 2 ** 32
    x = (torch.bitwise_xor(x, x // 2 ** 17) * 0xBB67AE85) % 2 ** 32
    return torch.bitwise_xor(x, x // 2 ** 15)


def _exact_block(s):
    x, h = s["x"].double(), s["h"].double()
    rows, d = x.shape
    gate = 1.0 if s["gate"] is None else s["gate"].double()[
        torch.arange(rows, device="cuda") * s["gate"].shape[0] // rows]
    rms_h = (h.pow(2).sum(1, keepdim=True) / d + s["eps"]).sqrt()
    y = s["residual_scale"] * x + s["branch_scale"] * gate * (h / rms_h * s["post_weight"].double())
    rms_y = (y.pow(2).sum(1, keepdim=True) / d + s["eps"]).sqrt()
    return {"y": y, "z": y / rms_y * s["pre_weight"].double(),
            "post_rstd": (1 / rms_h)[:, 0], "pre_rstd": (1 / rms_y)[:, 0]}


def _exact_block_grad(s):
    """The chain rule through z = y r w and y = a x + b gate (h q v), from the
    given y and statistics: d(r)/d(y) = -r^3 y / D."""
    y, h, dz, total = (s[k].double() for k in ("y", "h", "dz", "dy"))
    rows, d = y.shape
    owner = None if s["gate"] is None else (
        torch.arange(rows, device="cuda") * s["gate"].shape[0] // rows)
    gate = 1.0 if s["gate"] is None else s["gate"].double()[owner]
    w, v = s["pre_weight"].double(), s["post_weight"].double()
    r, q = s["pre_rstd"].double()[:, None], s["post_rstd"].double()[:, None]
    total = total + dz * w * r - y * r ** 3 / d * (dz * w * y).sum(1, keepdim=True)
    du = s["branch_scale"] * gate * total
    dh = du * v * q - h * q ** 3 / d * (du * v * h).sum(1, keepdim=True)
    dgate = None
    if s["gate"] is not None:
        dgate = torch.zeros(s["gate"].shape, dtype=torch.float64, device="cuda")
        dgate.index_add_(0, owner, s["branch_scale"] * total * h * q * v)
    return {"dx": s["residual_scale"] * total, "dh": dh, "dgate": dgate,
            "dpost_weight": (du * h * q).sum(0), "dpre_weight": (dz * y * r).sum(0)}
