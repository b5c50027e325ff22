"""block_norm and its gradients on the GPU against their 64-bit restatements:
types, widths, gates, strides, parts left out, streams, and refusals; and a
whole step of all the operators, eager and replayed from a graph."""

import numpy as np
import pytest
import torch

from oracle import train_oracle as o

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TYPES = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")]
WIDTHS = [1, 2, 7, 8, 63, 64, 250, 256, 264, 511, 512, 1000, 1023, 1024, 1032, 2048, 4096, 5001,
          8192, 8200, 9001, 16384, 16392, 32768, 32767]


@pytest.fixture(scope="module")
def ops():
    from loom_b200.build import load_train
    return load_train()


def dev(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda().to(DT[dtype])


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def half(dtype):
    return torch.finfo(DT[dtype]).eps / 2


def tiny(dtype):
    """Half the spacing of the type's smallest values."""
    return {"f32": 1e-45, "bf16": 1e-40, "f16": 2.0 ** -25}[dtype]


def near(got, want, err, dtype):
    """got: of `dtype`, within `err` of want before its own rounding."""
    got = f64(got).reshape(want.shape)
    bound = err + half(dtype) * (np.abs(want) + err) + tiny(dtype)
    worst = np.max(np.abs(got - want) - bound) if got.size else -1
    assert np.all(np.abs(got - want) <= bound), (worst, dtype)


def make(rows, width, tx, th, gate=None, strided=False, post=True, pre=True, has_h=True, seed=0):
    rng = np.random.default_rng(rows * 100003 + width + seed)
    s = {"x": dev(rng.normal(size=(rows, width)), tx), "h": None, "gate": None,
         "post_weight": None, "pre_weight": None}
    runs = {None: 0, "token": rows, "channel": 1}.get(gate, gate)
    if has_h:
        if strided:
            both = dev(rng.normal(size=(rows, 2 * width)), th)
            s["h"] = both[:, :width]
            if runs == rows:
                s["gate"] = both[:, width:]
            wide = torch.zeros(rows, width + 8, device="cuda", dtype=DT[tx])
            wide[:, 8:] = s["x"]
            s["x"] = wide[:, 8:]
        else:
            s["h"] = dev(rng.normal(size=(rows, width)) * 3, th)
        if runs and s["gate"] is None:
            s["gate"] = dev(rng.normal(size=(runs, width)), th)
        if post:
            s["post_weight"] = dev(1 + 0.2 * rng.normal(size=width), th)
    if pre:
        s["pre_weight"] = dev(1 + 0.2 * rng.normal(size=width), th)
    return s


def check_forward(ops, s, tx, th, post_norm=True, pre_norm=True, eps=1e-6, offset=0.0, a=1.0,
                  b=1.0, stream=None):
    got = ops["block_norm"](**s, post_norm=post_norm, pre_norm=pre_norm, eps=eps,
                            weight_offset=offset, residual_scale=a, branch_scale=b, stream=stream)
    torch.cuda.synchronize()
    n = {k: f64(v) for k, v in s.items()}
    y, z, q, r, parts = o.block_norm(n["x"], n["h"], n["gate"], n["post_weight"], n["pre_weight"],
                                     post_norm=post_norm, pre_norm=pre_norm, eps=eps,
                                     offset=offset, a=a, b=b)
    # a row's sum of squares: a thread adds at most 32 of them one by one and the
    # tree has at most 10 levels; nothing cancels, and the root halves it: 24 U with
    # the root's, the quotient's and the mean's own roundings
    err_q = 24 * o.U
    err_y = (err_q + 8 * o.U) * parts
    if q is not None:
        near(got.post_rstd, q, err_q * q, "f32")
    if s["h"] is not None:
        near(got.y, y, err_y, tx)
    else:
        assert got.y is s["x"]
        err_y = 0 * err_y
    if pre_norm:
        # y's errors move its norm by at most their own root mean square
        moved = np.sqrt(np.mean(err_y ** 2, axis=1, keepdims=True)) * r[:, None]
        near(got.pre_rstd, r, (err_q + moved[:, 0]) * r, "f32")
        scale = np.abs(r[:, None] * (1.0 if n["pre_weight"] is None else n["pre_weight"] + offset))
        near(got.z, z, scale * err_y + np.abs(z) * (err_q + moved + 6 * o.U), th)
    else:
        assert got.z is None and got.pre_rstd is None
    return got


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("tx,th", TYPES)
def test_forward_widths(ops, width, tx, th):
    check_forward(ops, make(5, width, tx, th, gate="token"), tx, th)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 149, 1000])
@pytest.mark.parametrize("width", [64, 1000, 4096])
def test_forward_rows(ops, rows, width):
    check_forward(ops, make(rows, width, "bf16", "bf16"), "bf16", "bf16")


@pytest.mark.parametrize("width", [104, 249, 257, 264, 1023, 2048, 5001, 8200, 20000])
@pytest.mark.parametrize("tx,th", TYPES)
@pytest.mark.parametrize("gate", [None, "token", 6])
def test_forward_several_rows_a_group(ops, width, tx, th, gate):
    """More rows than the SMs hold at once, so that row groups walk several."""
    rows = 6 * (1100 if width < 256 else 500 if width < 1100 else 110)
    check_forward(ops, make(rows, width, tx, th, gate=gate), tx, th)


@pytest.mark.parametrize("gate", [None, "token", "channel", 2, 3])
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("width", [96, 257, 2048])
def test_forward_gates_and_strides(ops, gate, strided, width):
    check_forward(ops, make(12, width, "f32", "bf16", gate=gate, strided=strided), "f32", "bf16",
                  offset=1.0, a=0.5, b=-2.0, eps=1e-2)


@pytest.mark.parametrize("form", ["no h", "no post norm", "no pre norm", "no weights",
                                  "no norms", "no gate or weights"])
@pytest.mark.parametrize("width", [100, 1024, 1536])
def test_forward_parts_left_out(ops, form, width):
    kw, flags = {}, {}
    if form == "no h":
        kw = dict(has_h=False)
    elif form == "no post norm":
        kw, flags = dict(post=False, gate="token"), dict(post_norm=False)
    elif form == "no pre norm":
        kw, flags = dict(pre=False, gate="token"), dict(pre_norm=False)
    elif form == "no norms":
        kw, flags = dict(post=False, pre=False, gate="channel"), dict(post_norm=False,
                                                                      pre_norm=False)
    elif form == "no weights":
        kw = dict(post=False, pre=False, gate="channel")
    else:
        kw = dict(post=False, pre=False)
    check_forward(ops, make(7, width, "bf16", "bf16", **kw), "bf16", "bf16", offset=0.5, **flags)


def test_rows_of_zeros_and_of_values_that_are_not_finite(ops):
    """A row of zeros has the statistic of eps; a row that holds NaN or
    infinity leaves the other rows alone."""
    s = make(6, 1024, "f32", "f32")
    clean = ops["block_norm"](**s)
    s["h"][1] = 0
    s["x"][1] = 0
    s["h"][3, 17] = float("inf")
    s["x"][4, 5] = float("nan")
    got = ops["block_norm"](**s)
    # 1 / sqrt(1e-6): the root's and the quotient's roundings, and eps's own
    assert abs(float(got.post_rstd[1]) - 1000) < 3 * o.U * 1000
    assert torch.all(got.z[1] == 0) and torch.all(got.y[1] == 0)
    assert torch.isnan(got.z[4]).all()
    for row in (0, 2, 5):
        assert torch.equal(got.z[row], clean.z[row]) and torch.equal(got.y[row], clean.y[row])


def padded(t, pad=8):
    """The same rows at a stride of `pad` more, NaN between them and behind them."""
    rows, width = t.shape
    wide = torch.full((rows, width + pad), float("nan"), device="cuda").to(t.dtype)
    wide[:, :width] = t
    return wide[:, :width]


@pytest.mark.parametrize("width", [25, 257, 1023, 1536])
@pytest.mark.parametrize("tx,th", [("bf16", "bf16"), ("f32", "f16")])
def test_what_lies_between_rows_stays_out(ops, width, tx, th):
    """Odd widths' groups reach into the row before: rows with NaN between them,
    and a row of NaN among the others, in both directions."""
    rows = 2400 if width < 256 else 1700
    s = make(rows, width, tx, th, gate="token")
    wide = {k: padded(v) if k in ("x", "h", "gate") else v for k, v in s.items()}
    want, got = ops["block_norm"](**s), ops["block_norm"](**wide)
    assert torch.equal(got.y, want.y) and torch.equal(got.z, want.z)
    rest = {k: v for k, v in s.items() if k != "x"}
    stats = dict(post_rstd=want.post_rstd, pre_rstd=want.pre_rstd)
    grads = ops["block_norm_backward"](y=want.y, dy=want.y, dz=want.z, **stats, **rest)
    rest = {k: v for k, v in wide.items() if k != "x"}
    again = ops["block_norm_backward"](y=padded(want.y), dy=padded(want.y), dz=padded(want.z),
                                       **stats, **rest)
    for a, b in zip(again, grads):
        assert torch.equal(a, b)
    bad = 7
    s["h"][bad] = float("nan")
    got = ops["block_norm"](**s)
    others = torch.arange(rows, device="cuda") != bad
    assert torch.isnan(got.z[bad]).all()
    assert torch.equal(got.z[others], want.z[others]) and torch.equal(got.y[others],
                                                                      want.y[others])
    rest = {k: v for k, v in s.items() if k != "x"}
    bad_grads = ops["block_norm_backward"](y=got.y, dy=want.y, dz=want.z,
                                           post_rstd=got.post_rstd, pre_rstd=got.pre_rstd, **rest)
    assert torch.equal(bad_grads.dx[others], grads.dx[others])
    assert torch.equal(bad_grads.dh[others], grads.dh[others])
    assert torch.equal(bad_grads.dgate[others], grads.dgate[others])


def test_an_output_given_twice_is_refused(ops):
    s = make(12, 64, "f32", "f32")
    out = ops["block_norm"](**s)
    with pytest.raises(ValueError):
        ops["block_norm"](**s, out=out._replace(pre_rstd=out.post_rstd))
    with pytest.raises(ValueError):
        ops["block_norm"](**s, out=out._replace(z=out.y))
    ops["block_norm"](**s, out=out)


def test_shapes_and_given_outputs(ops):
    s = make(12, 64, "f32", "bf16", gate=3)
    flat = ops["block_norm"](**s)
    t = {k: v.view(3, 4, 64) if k in ("x", "h") else v for k, v in s.items()}
    t["gate"] = s["gate"].view(3, 1, 64)
    out = type(flat)(torch.empty(3, 4, 64, device="cuda"),
                     torch.empty(3, 4, 64, device="cuda", dtype=torch.bfloat16),
                     torch.empty(12, device="cuda"), torch.empty(12, device="cuda"))
    got = ops["block_norm"](**t, out=out)
    assert got.y is out.y and got.z is out.z
    assert torch.equal(got.y.view(12, 64), flat.y) and torch.equal(got.z.view(12, 64), flat.z)
    empty = ops["block_norm"](x=s["x"][:0], h=s["h"][:0], pre_weight=s["pre_weight"])
    assert empty.y.shape == (0, 64) and empty.z.shape == (0, 64)


# ---------------------------------------------------------------------------
# gradients


def check_backward(ops, s, tx, th, post_norm=True, pre_norm=True, offset=0.0, a=1.0, b=1.0,
                   with_dy=True, stream=None, seed=0):
    rows, width = s["x"].shape
    n = {k: f64(v) for k, v in s.items()}
    y, _, q, r, _ = o.block_norm(n["x"], n["h"], n["gate"], n["post_weight"], n["pre_weight"],
                                 post_norm=post_norm, pre_norm=pre_norm, offset=offset, a=a, b=b)
    rng = np.random.default_rng(rows + 7 * width + seed)
    given = {"y": dev(y, tx) if s["h"] is not None else s["x"],
             "post_rstd": None if q is None else dev(q, "f32"),
             "pre_rstd": None if r is None else dev(r, "f32"),
             "dy": dev(rng.normal(size=(rows, width)), tx) if with_dy else None,
             "dz": dev(rng.normal(size=(rows, width)), th) if pre_norm else None}
    call = {k: v for k, v in s.items() if k != "x"}
    got = ops["block_norm_backward"](**given, **call, post_norm=post_norm, pre_norm=pre_norm,
                                     weight_offset=offset, residual_scale=a, branch_scale=b,
                                     stream=stream)
    torch.cuda.synchronize()
    g = {k: f64(v) for k, v in given.items()}
    want = o.block_norm_grads(g["y"], n["h"], n["gate"], n["post_weight"], n["pre_weight"],
                              g["post_rstd"], g["pre_rstd"], g["dy"], g["dz"], offset=offset, a=a,
                              b=b)
    # an element: two row sums of at most 32 + 10 additions each, and their products;
    # a sum over rows: as many additions again as it has rows
    own = 110 * o.U
    for name in ("dx", "dh", "dgate", "dpost_weight", "dpre_weight"):
        t = getattr(got, name)
        if name not in want or (name == "dpost_weight" and s["post_weight"] is None) or (
                name == "dpre_weight" and s["pre_weight"] is None):
            assert t is None, name
            continue
        value, size = want[name]
        along = {"dx": 0, "dh": 0,
                 "dgate": 0 if s["gate"] is None else rows // max(1, s["gate"].shape[0])}
        near(t, value, (own + along.get(name, rows) * o.U) * size,
             tx if name == "dx" else th)
    return got


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("tx,th", TYPES)
def test_backward_widths(ops, width, tx, th):
    check_backward(ops, make(5, width, tx, th, gate="token"), tx, th)


@pytest.mark.parametrize("rows", [1, 2, 3, 300, 1500])
@pytest.mark.parametrize("width", [64, 1000, 2048])
def test_backward_rows(ops, rows, width):
    check_backward(ops, make(rows, width, "f32", "f32"), "f32", "f32")


@pytest.mark.parametrize("gate", [None, "token", "channel", 2, 6, 120])
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("width", [96, 257, 2048])
def test_backward_gates_and_strides(ops, gate, strided, width):
    check_backward(ops, make(600, width, "f32", "bf16", gate=gate, strided=strided), "f32", "bf16",
                   offset=1.0, a=0.5, b=-2.0)


@pytest.mark.parametrize("width", [249, 256, 1536, 4096, 4100, 6144, 8192, 8191])
@pytest.mark.parametrize("tx,th", [("f32", "f32"), ("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("gate", [None, "token", "channel", 4])
def test_backward_several_rows_a_group(ops, width, tx, th, gate):
    check_backward(ops, make(2080 if width == 4096 else 640, width, tx, th, gate=gate), tx, th,
                   b=0.5, seed=3)


@pytest.mark.parametrize("runs", [1500, 750, 300, 1])
def test_backward_many_gate_rows(ops, runs):
    check_backward(ops, make(1500, 264, "f16", "f16", gate=runs), "f16", "f16")


@pytest.mark.parametrize("form", ["no h", "no post norm", "no pre norm", "no weights", "no dy",
                                  "no norms"])
@pytest.mark.parametrize("width", [100, 1024, 1536])
def test_backward_parts_left_out(ops, form, width):
    kw, flags = dict(gate="token"), {}
    if form == "no h":
        kw = dict(has_h=False)
    elif form == "no post norm":
        kw, flags = dict(post=False, gate=3), dict(post_norm=False)
    elif form == "no pre norm":
        kw, flags = dict(pre=False, gate="token"), dict(pre_norm=False)
    elif form == "no norms":
        kw, flags = dict(post=False, pre=False, gate="channel"), dict(post_norm=False,
                                                                      pre_norm=False)
    elif form == "no weights":
        kw = dict(post=False, pre=False)
    else:
        flags = dict(with_dy=False)
    check_backward(ops, make(9, width, "bf16", "bf16", **kw), "bf16", "bf16", offset=0.5, **flags)


@pytest.mark.parametrize("width", [100, 1023, 1024, 9001])
@pytest.mark.parametrize("tx,th", [("f32", "f32"), ("f32", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("rows", [9, 700])
def test_without_h_the_residual_scale_has_no_part(ops, width, tx, th, rows):
    s = make(rows, width, tx, th, has_h=False)
    check_forward(ops, s, tx, th, a=0.7, b=3.0, offset=0.5)
    got = check_backward(ops, s, tx, th, a=0.7, b=3.0, offset=0.5)
    plain = check_backward(ops, s, tx, th, offset=0.5)
    assert torch.equal(got.dx, plain.dx) and torch.equal(got.dpre_weight, plain.dpre_weight)


@pytest.mark.parametrize("gate", [None, "token", "channel", 5])
@pytest.mark.parametrize("width", [100, 1024, 1023])
@pytest.mark.parametrize("rows", [10, 900])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_without_norms_dh_does_not_hang_on_h(ops, gate, width, rows, bad):
    """y = a x + b gate h: a value of h that is not finite stays out of dh and dx."""
    s = make(rows, width, "bf16", "bf16", gate=gate, post=False, pre=False)
    dy = dev(np.random.default_rng(5).normal(size=(rows, width)), "bf16")
    call = dict(y=s["x"], dy=dy, gate=s["gate"], post_norm=False, pre_norm=False,
                residual_scale=0.5, branch_scale=2.0)
    want = ops["block_norm_backward"](h=s["h"], **call)
    s["h"][3, 7] = bad
    got = ops["block_norm_backward"](h=s["h"], **call)
    assert torch.equal(got.dh, want.dh) and torch.equal(got.dx, want.dx)
    if gate == "token":  # each gate row's gradient has one row of h
        assert not torch.isfinite(got.dgate[3, 7])
        got.dgate[3, 7] = want.dgate[3, 7]
        assert torch.equal(got.dgate, want.dgate)
    n = {k: f64(v) for k, v in s.items()}
    runs = 1.0 if gate is None else np.repeat(n["gate"], rows // n["gate"].shape[0], axis=0)
    near(got.dh, 2.0 * runs * f64(dy), 3 * o.U * np.abs(2.0 * runs * f64(dy)), "bf16")


def test_backward_of_no_rows(ops):
    s = make(6, 64, "f32", "f32", gate="channel")
    none = {k: (v[:0] if k in ("x", "h") else v) for k, v in s.items()}
    call = {k: v for k, v in none.items() if k != "x"}
    e = torch.empty(0, device="cuda")
    got = ops["block_norm_backward"](y=none["x"], dy=none["x"], dz=none["x"], post_rstd=e,
                                     pre_rstd=e, **call)
    assert got.dx.shape == (0, 64) and torch.all(got.dgate == 0)
    assert torch.all(got.dpre_weight == 0) and torch.all(got.dpost_weight == 0)


def test_backward_is_the_same_every_time(ops):
    s = make(1000, 1024, "bf16", "bf16", gate="channel")
    got = [check_backward(ops, s, "bf16", "bf16") for _ in range(3)]
    for g in got[1:]:
        for a, b in zip(g, got[0]):
            assert torch.equal(a, b)


def test_gradients_against_differences_of_the_kernels(ops):
    """The kernels' own forward pass, moved along a direction, against the
    product of its gradients with that direction."""
    s = make(40, 320, "f32", "f32", gate=4)
    rng = np.random.default_rng(2)
    cy, cz = (dev(rng.normal(size=(40, 320)), "f32") for _ in range(2))
    names = {"x": "dx", "h": "dh", "gate": "dgate", "post_weight": "dpost_weight",
             "pre_weight": "dpre_weight"}
    direction = {k: dev(rng.normal(size=tuple(v.shape)), "f32") for k, v in s.items()}
    out = ops["block_norm"](**s, branch_scale=0.7)
    grads = ops["block_norm_backward"](
        y=out.y, post_rstd=out.post_rstd, pre_rstd=out.pre_rstd, dy=cy, dz=cz, branch_scale=0.7,
        **{k: v for k, v in s.items() if k != "x"})

    def value(step, key):
        moved = {k: v + step * direction[k] if k == key else v for k, v in s.items()}
        r = ops["block_norm"](**moved, branch_scale=0.7)
        return float((cy.double() * r.y.double()).sum() + (cz.double() * r.z.double()).sum())

    for key, name in names.items():
        step = 2.0 ** -7
        # fourth-order differences: the remaining error is of order step^4
        slope = (8 * (value(step, key) - value(-step, key))
                 - (value(2 * step, key) - value(-2 * step, key))) / (12 * step)
        got = float((getattr(grads, name).double() * direction[key].double()).sum())
        size = float((getattr(grads, name).double() * direction[key].double()).abs().sum())
        # the forward values' roundings are independent: about U times the root of
        # 25600 terms of order 3 over the step, 0.004; and the fourth-order term,
        # 4 step^4 of the terms' size, 1.5e-8 of it times the fifth derivative's weight
        assert abs(slope - got) < 0.02 + 1e-4 * size ** 0.5 + 1e-6 * size, (key, slope, got)


# ---------------------------------------------------------------------------
# streams, graphs and a whole step


def test_side_streams_side_by_side(ops):
    sets = [make(300, 1024, "bf16", "bf16", gate="token", seed=i) for i in range(3)]
    alone = [ops["block_norm"](**s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(3):
        got = [ops["block_norm"](**s, stream=st) for s, st in zip(sets, streams)]
    torch.cuda.synchronize()
    for g, a in zip(got, alone):
        assert torch.equal(g.z, a.z) and torch.equal(g.y, a.y)


class Step:
    """One training step of a block's norm weights and gate: forward, backward,
    the gradients' norm, and an AdamW step that takes its factor."""

    def __init__(self, ops, eight, stream):
        rows, width = 200, 512
        s = make(rows, width, "bf16", "bf16", gate="channel", seed=4)
        self.s = s
        rng = np.random.default_rng(1)
        dy, dz = (dev(rng.normal(size=(rows, width)), "bf16") for _ in range(2))
        self.params = [s["gate"], s["post_weight"], s["pre_weight"]]
        f = ops["block_norm"].bind(stream=stream, **s)
        b = ops["block_norm_backward"].bind(
            stream=stream, y=f[1].y, post_rstd=f[1].post_rstd, pre_rstd=f[1].pre_rstd, dy=dy,
            dz=dz, **{k: v for k, v in s.items() if k != "x"})
        grads = [b[1].dgate, b[1].dpost_weight, b[1].dpre_weight]
        n = ops["grad_norm"].bind(stream=stream, grads=grads, max_norm=1.0)
        self.norm = n[1]
        sizes = [p.numel() for p in self.params]
        new = lambda d, ns: [torch.zeros(k, device="cuda").to(d) for k in ns]  # noqa: E731
        self.step = torch.zeros(1, dtype=torch.int64, device="cuda")
        self.lr = torch.tensor([1e-2], device="cuda")
        self.master = [p.float() for p in self.params]
        kind = torch.float8_e4m3fn if eight else torch.float32
        self.m, self.v = new(kind, sizes), new(kind, sizes)
        more = {}
        if eight:
            tops = [-(-k // 256) for k in sizes]
            self.tops = new(torch.float32, tops) + new(torch.float32, tops)
            more = dict(exp_avg_top=self.tops[:3], exp_avg_sq_top=self.tops[3:], seed=77)
        u = ops["adamw8" if eight else "adamw"].bind(
            stream=stream, params=self.params, grads=grads, exp_avg=self.m, exp_avg_sq=self.v,
            master=self.master, step=self.step, lr=self.lr, weight_decay=[0.0, 0.1, 0.1],
            betas=(0.9, 0.95), grad_scale=self.norm[1:], **more)
        self.calls = [c for c, _ in (f, b, n, u)]

    def __call__(self):
        for c in self.calls:
            c()

    def state(self):
        return [t.view(torch.uint8).clone() for t in
                self.params + self.master + self.m + self.v + [self.step, self.norm]]


@pytest.mark.parametrize("eight", [False, True])
def test_a_whole_step_eager_and_replayed(ops, eight):
    side = torch.cuda.Stream()
    eager, graphed = Step(ops, eight, side), Step(ops, eight, side)
    torch.cuda.synchronize()
    before = eager.params[1].clone()
    with torch.cuda.stream(side):
        for _ in range(5):
            eager()
    torch.cuda.synchronize()
    assert not torch.equal(eager.params[1], before) and int(eager.step) == 5
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        graphed()
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(eager.state(), graphed.state()):
        assert torch.equal(a, b)
    # the learning rate is read at replay: a rate of zero leaves the masters, but for decay
    graphed.lr.zero_()
    kept = [t.clone() for t in graphed.master]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, graphed.master))
    assert int(graphed.step) == 6


def test_host_threads_with_rows_of_two_widths(ops):
    """Two threads' launches of one kernel whose rows take different amounts of
    shared memory: neither may lower what the other has asked for."""
    import threading
    sets = [make(1200, width, "bf16", "bf16", gate="token") for width in (2048, 4096)]
    want, calls, outs = [], [], []
    for s in sets:
        out = ops["block_norm"](**s)
        back = dict(y=out.y, post_rstd=out.post_rstd, pre_rstd=out.pre_rstd, dy=out.y, dz=out.z,
                    **{k: v for k, v in s.items() if k != "x"})
        want.append(list(out) + list(ops["block_norm_backward"](**back)))
        stream = torch.cuda.Stream()
        f = ops["block_norm"].bind(stream=stream, **s)
        b = ops["block_norm_backward"].bind(stream=stream, **back)
        calls.append((f[0], b[0]))
        outs.append(list(f[1]) + list(b[1]))
    torch.cuda.synchronize()
    errors, gate = [], threading.Barrier(2)

    def many(pair):
        try:
            gate.wait(timeout=60)
            for _ in range(1500):
                for call in pair:
                    call()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=many, args=(pair,)) for pair in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for got, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_a_graph_of_two_widths(ops):
    """One graph holds launches of one kernel with two amounts of shared memory;
    eager calls of the smaller one come between its replays."""
    sets = [make(1200, width, "bf16", "bf16", gate="token") for width in (4096, 2048)]
    want = [ops["block_norm"](**s) for s in sets]
    side = torch.cuda.Stream()
    bound = [ops["block_norm"].bind(stream=side, **s) for s in sets]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for call, _ in bound:
            call()
    for _ in range(3):
        ops["block_norm"](**sets[1])
        for _, out in bound:
            out.y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for (_, out), w in zip(bound, want):
            assert torch.equal(out.y, w.y) and torch.equal(out.z, w.z)


def test_two_graphs_of_two_bindings_side_by_side(ops):
    """Two graphs, replayed on two streams at once: each binding has a
    workspace of its own."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = [make(500, 1024, "bf16", "bf16", gate="channel", seed=i) for i in range(2)]
    want, bound, graphs = [], [], []
    for s, st in zip(sets, streams):
        out = ops["block_norm"](**s)
        args = dict(y=out.y, post_rstd=out.post_rstd, pre_rstd=out.pre_rstd, dy=out.y, dz=out.z,
                    **{k: v for k, v in s.items() if k != "x"})
        want.append(ops["block_norm_backward"](**args))
        torch.cuda.synchronize()
        bound.append(ops["block_norm_backward"].bind(stream=st, **args))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            bound[-1][0]()
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (_, got), w in zip(bound, want):
        for a, b in zip(got, w):
            assert torch.equal(a, b)


def test_calls_inside_a_capture_allocate_their_own(ops):
    """Direct calls under capture take their outputs and workspaces from the
    graph's memory."""
    s = make(64, 768, "f32", "bf16", gate="channel")
    want = ops["block_norm"](**s)
    grads = ops["block_norm_backward"](y=want.y, post_rstd=want.post_rstd, pre_rstd=want.pre_rstd,
                                       dy=want.y, dz=want.z,
                                       **{k: v for k, v in s.items() if k != "x"})
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out = ops["block_norm"](**s, stream=side)
        got = ops["block_norm_backward"](y=out.y, post_rstd=out.post_rstd, pre_rstd=out.pre_rstd,
                                         dy=out.y, dz=out.z, stream=side,
                                         **{k: v for k, v in s.items() if k != "x"})
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, grads):
        assert torch.equal(a, b)


def test_refusals(ops):
    s = make(12, 64, "bf16", "bf16", gate=3)
    f = ops["block_norm"]
    for change, error in [
            (dict(h=s["h"].float()), TypeError), (dict(h=s["h"][:6]), ValueError),
            (dict(gate=s["gate"].expand(3, 64)[:, :63]), ValueError),
            (dict(gate=torch.ones(5, 64, device="cuda", dtype=torch.bfloat16)), ValueError),
            (dict(post_weight=s["post_weight"][:63]), ValueError),
            (dict(pre_weight=s["pre_weight"].float()), TypeError),
            (dict(pre_norm=False), ValueError), (dict(post_norm=False), ValueError),
            (dict(h=None), ValueError), (dict(eps=-1.0), ValueError),
            (dict(eps=float("nan")), ValueError), (dict(branch_scale=float("inf")), ValueError),
            (dict(h=s["h"].t().contiguous().t()), ValueError),
            (dict(x=s["x"].double()), TypeError),
            (dict(x=torch.zeros(2, 32769, device="cuda")), ValueError),
            (dict(x=torch.zeros(2, 0, device="cuda")), ValueError)]:
        with pytest.raises(error):
            f(**{**s, **change})
    out = f(**s)
    with pytest.raises(ValueError):
        f(**s, out=out._replace(y=s["x"]))
    with pytest.raises(ValueError):
        f(**s, out=out._replace(z=out.z[:6]))
    g = ops["block_norm_backward"]
    good = dict(y=out.y, post_rstd=out.post_rstd, pre_rstd=out.pre_rstd, dy=out.y, dz=out.z,
                **{k: v for k, v in s.items() if k != "x"})
    for change, error in [(dict(dz=None), ValueError), (dict(pre_rstd=None), ValueError),
                          (dict(post_rstd=out.post_rstd[:5]), ValueError),
                          (dict(dy=out.y.float()), TypeError), (dict(dy=out.y[:3]), ValueError)]:
        with pytest.raises(error):
            g(**{**good, **change})


def test_numbers_beyond_fp32_and_rows_beyond_31_bits_are_refused(ops):
    """Before anything runs, as ValueError: the C entries take floats."""
    s = make(12, 64, "bf16", "bf16")
    for change in (dict(eps=1e39), dict(eps=float("inf")), dict(residual_scale=1e39),
                   dict(branch_scale=-4e38), dict(weight_offset=float("nan"))):
        with pytest.raises(ValueError):
            ops["block_norm"](**{**s, **change})
    # rows that share one place in memory: nothing of this size is allocated
    many = torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16).expand(1 << 31, 1)
    with pytest.raises(ValueError):
        ops["block_norm"](x=many)
    with pytest.raises(ValueError):
        ops["block_norm_backward"](y=many, dz=many, pre_rstd=many)
    far = torch.empty((1 << 31) + 8, device="cuda", dtype=torch.bfloat16).as_strided(
        (2, 8), (1 << 31, 1))
    with pytest.raises(ValueError):
        ops["block_norm"](x=far)
    with pytest.raises(ValueError):
        ops["block_norm"](x=far[:1].expand(2, 8), h=far)


def test_offsets_beyond_31_bits(ops):
    """Rows so far apart that elements' places pass 2^31, in both directions."""
    rows, width, apart = 40, 264, 100_000_000
    s = make(rows, width, "bf16", "bf16", gate="token")
    wide = {}
    for k in ("x", "h", "gate"):
        buf = torch.empty((rows - 1) * apart + width, device="cuda", dtype=torch.bfloat16)
        wide[k] = buf.as_strided((rows, width), (apart, 1))
        wide[k].copy_(s[k])
    want = ops["block_norm"](**s)
    got = ops["block_norm"](**{**s, **wide})
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    rest = dict(post_weight=s["post_weight"], pre_weight=s["pre_weight"], dy=want.y, dz=want.z,
                post_rstd=want.post_rstd, pre_rstd=want.pre_rstd)
    grads = ops["block_norm_backward"](y=want.y, h=s["h"], gate=s["gate"], **rest)
    again = ops["block_norm_backward"](y=wide["x"].copy_(want.y), h=wide["h"], gate=wide["gate"],
                                       **rest)
    for a, b in zip(again, grads):
        assert torch.equal(a, b)


def test_many_rows_with_outputs_beyond_31_bits(ops):
    """More than 2^31 elements, contiguous: the last rows are those of a short call."""
    width, rows = 4096, (1 << 19) + 4096
    x = torch.zeros(rows, width, device="cuda", dtype=torch.bfloat16)
    s = make(4096, width, "bf16", "bf16", has_h=False)
    x[-4096:] = s["x"]
    want = ops["block_norm"](x=s["x"], pre_weight=s["pre_weight"])
    got = ops["block_norm"](x=x, pre_weight=s["pre_weight"])
    assert torch.equal(got.z[-4096:], want.z) and not got.z[:-4096].any()
    assert torch.equal(got.pre_rstd[-4096:], want.pre_rstd)
    dz = torch.zeros_like(x)
    dz[-4096:] = want.z
    grads = ops["block_norm_backward"](y=s["x"], pre_weight=s["pre_weight"], dz=want.z,
                                       pre_rstd=want.pre_rstd)
    again = ops["block_norm_backward"](y=x, pre_weight=s["pre_weight"], dz=dz,
                                       pre_rstd=got.pre_rstd)
    assert torch.equal(again.dx[-4096:], grads.dx) and not again.dx[:-4096].any()


def placed(t, first=1, gap=0):
    """The same rows `first` elements behind a 16-byte boundary, `gap` apart; NaN
    around them."""
    t2 = t if t.dim() == 2 else t[None]
    rows, width = t2.shape
    stride = width + gap
    buf = torch.full((first + rows * stride + 8,), float("nan"), device="cuda").to(t.dtype)
    v = buf[first:].as_strided((rows, width), (stride, 1))
    v.copy_(t2)
    return v if t.dim() == 2 else v[0]


@pytest.mark.parametrize("first,gap", [(1, 0), (3, 5), (8, 1), (0, 13)])
@pytest.mark.parametrize("gate", [None, "token", 3])
@pytest.mark.parametrize("width", [1, 40, 257, 1024, 4096, 8200])
@pytest.mark.parametrize("tx,th", [("bf16", "bf16"), ("f32", "f16")])
def test_rows_at_any_place(ops, width, tx, th, gate, first, gap):
    """Bases and distances of every alignment, given outputs too, against the same
    rows at a boundary: within the roundings of sums in another order."""
    rows = 600 if width < 1000 else 18
    s = make(rows, width, tx, th, gate=gate)
    moved = {k: v if v is None else placed(v, first, gap) for k, v in s.items()}
    check_forward(ops, moved, tx, th, b=0.5)
    check_backward(ops, moved, tx, th, b=0.5)
    want = ops["block_norm"](**s, branch_scale=0.5)
    out = type(want)(*[placed(torch.zeros_like(t), first) for t in want])
    got = ops["block_norm"](**moved, branch_scale=0.5, out=out)
    clean = ops["block_norm"](**moved, branch_scale=0.5)
    for a, b in zip(got, clean):
        # the outputs' places may choose another kernel: two orders of the fp32 sums
        near(a, f64(b), 60 * o.U * np.maximum(1.0, np.abs(f64(b))),
             {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}[a.dtype])
    n = {k: f64(v) for k, v in s.items()}
    rng = np.random.default_rng(width)
    dy, dz = dev(rng.normal(size=(rows, width)), tx), dev(rng.normal(size=(rows, width)), th)
    call = dict(post_rstd=want.post_rstd, pre_rstd=want.pre_rstd, branch_scale=0.5)
    got = ops["block_norm_backward"](
        y=placed(want.y, first, gap), dy=placed(dy, first, gap), dz=placed(dz, first, gap),
        **{k: v for k, v in moved.items() if k != "x"}, **call)
    exact = o.block_norm_grads(f64(want.y), n["h"], n["gate"], n["post_weight"], n["pre_weight"],
                               f64(want.post_rstd), f64(want.pre_rstd), f64(dy), f64(dz), b=0.5)
    for name, (value, size) in exact.items():   # bounds as in check_backward
        along = {"dx": 0, "dh": 0, "dgate": 0 if gate is None else rows // s["gate"].shape[0]}
        near(getattr(got, name), value, (110 + along.get(name, rows)) * o.U * size,
             tx if name == "dx" else th)


@pytest.mark.parametrize("width", [40, 257, 1024])
def test_rows_that_share_memory(ops, width):
    """Expanded inputs: every row of x, of the gate and of dy is one row."""
    s = make(30, width, "f32", "f32", gate="token")
    for k in ("x", "gate"):
        s[k] = s[k][:1].expand(30, width)
    full = {k: v.contiguous() for k, v in s.items()}
    got, want = ops["block_norm"](**s), ops["block_norm"](**full)
    check_forward(ops, s, "f32", "f32")
    check_backward(ops, s, "f32", "f32")
    near(got.z, f64(want.z), 60 * o.U * np.maximum(1.0, np.abs(f64(want.z))), "f32")
    dy = s["x"]
    call = dict(dz=want.z, post_rstd=want.post_rstd, pre_rstd=want.pre_rstd, y=want.y)
    a = ops["block_norm_backward"](dy=dy, **{k: v for k, v in s.items() if k != "x"}, **call)
    assert a.dgate.shape == (30, width) and a.dgate.is_contiguous()
    b = ops["block_norm_backward"](dy=dy.contiguous(),
                                   **{k: v for k, v in full.items() if k != "x"}, **call)
    for u, v in zip(a, b):
        near(u, f64(v), 200 * o.U * np.maximum(8.0, np.abs(f64(v))), "f32")


def test_three_dimensions_and_streams_by_handle(ops):
    """The halves of a projection in three dimensions, on streams given as handles."""
    both = dev(np.random.default_rng(3).normal(size=(3, 20, 512)), "bf16")
    x = dev(np.random.default_rng(4).normal(size=(3, 20, 256)), "bf16").requires_grad_()
    w = torch.ones(256, device="cuda", dtype=torch.bfloat16)
    a = dict(x=x, h=both[..., :256], gate=both[..., 256:], post_weight=w, pre_weight=w)
    want = ops["block_norm"](**{k: v.detach().reshape(-1, v.shape[-1]) if v.dim() == 3 else v
                                for k, v in a.items()})
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (None, 0, side, side.cuda_stream, torch.cuda.current_stream()):
        got = ops["block_norm"](**a, stream=stream)
        call, out = ops["block_norm"].bind(**a, stream=stream)
        call()
        torch.cuda.synchronize()
        for t in (got, out):
            assert t.y.shape == (3, 20, 256) and t.pre_rstd.shape == (60,)
            assert torch.equal(t.z.view(-1, 256), want.z) and torch.equal(t.y.view(-1, 256), want.y)
