"""The operators over lists of tensors on the GPU against their 64-bit
restatements: types, odd sizes, misaligned and empty tensors, long lists,
skipped steps, what lies around the tensors, streams and refusals."""

import numpy as np
import pytest
import torch

from oracle import train_oracle as o

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HYPER = dict(beta1=0.9, beta2=0.95, eps=1e-8)


@pytest.fixture(scope="module")
def ops():
    from loom_b200.build import load_train
    return load_train()


def guarded(values, dtype, offset=0, pad=64):
    """A device tensor of these values inside a larger buffer whose other
    elements have a value of their own; returns (view, buffer, check)."""
    n = len(values)
    buf = torch.full((pad + offset + n + pad,), 7.0, device="cuda").to(dtype)
    view = buf[pad + offset:pad + offset + n]
    view.copy_(torch.as_tensor(np.asarray(values), device="cuda"))

    def untouched():
        rest = torch.cat([buf[:pad + offset], buf[pad + offset + n:]]).float()
        return bool((rest == torch.tensor(7.0).to(dtype).float()).all())
    return view, untouched


def host(t):
    return t.detach().float().cpu().numpy()


# ---------------------------------------------------------------------------
# grad_norm

SIZE_LISTS = [[1], [3], [1024], [4097, 1, 0, 8191], [0, 5, 0], [70001, 16384, 255, 8192, 33],
              [1 << 20, 12345]]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("sizes", SIZE_LISTS, ids=str)
@pytest.mark.parametrize("offset", [0, 1, 5])
def test_norm_matches(ops, dtype, sizes, offset):
    rng = np.random.default_rng(sum(sizes) + offset)
    views = [guarded(rng.normal(size=n) * 10.0 ** rng.uniform(-3, 1), DT[dtype], offset)[0]
             for n in sizes]
    want, factor = o.norm_and_factor([host(v) for v in views], 0.5)
    got = ops["grad_norm"](grads=views, max_norm=0.5).cpu().numpy().astype(np.float64)
    # fp32 squares and at most 6 fp32 additions of values that do not cancel, half of
    # which passes on to the root, and the result's own rounding: (7 / 2 + 1) U
    assert abs(got[0] - want) <= 4.5 * o.U * want
    assert abs(got[1] - factor) <= 5.5 * o.U * factor


def test_norm_of_a_long_list_and_of_nothing(ops):
    rng = np.random.default_rng(1)
    grads = [torch.from_numpy(rng.normal(size=int(n)).astype(np.float32)).cuda()
             for n in rng.integers(0, 300, size=2500)]
    want, _ = o.norm_and_factor([host(g) for g in grads], 1.0)
    got = ops["grad_norm"](grads=grads, max_norm=float("inf")).cpu().numpy()
    assert abs(float(got[0]) - want) <= 4.5 * o.U * want and got[1] == 1.0
    empty = [torch.empty(0, device="cuda")]
    assert ops["grad_norm"](grads=empty, max_norm=1.0).cpu().tolist() == [0.0, 1.0]


@pytest.mark.parametrize("bad,norm", [(float("inf"), "inf"), (float("nan"), "nan"),
                                      (3e38, "inf")])
@pytest.mark.parametrize("place", [0, 5000, 99999])
def test_norm_of_values_that_are_not_finite(ops, bad, norm, place):
    g = torch.ones(100000, device="cuda")
    g[place] = bad
    got = ops["grad_norm"](grads=[torch.ones(3, device="cuda"), g], max_norm=1.0).cpu().numpy()
    assert np.isnan(got[1])
    assert np.isinf(got[0]) if norm == "inf" else np.isnan(got[0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e-20, 1e-22, 1e-25, 1e-36, 3e18, 1.2e19])
@pytest.mark.parametrize("offset", [0, 3])
def test_norm_of_squares_outside_the_fp32_range(ops, dtype, size, offset):
    """Squares below the fp32 range, and finite ones whose sum passes it: whole
    tiles, partial ones and ragged ends."""
    rng = np.random.default_rng(12)
    views = [guarded(size * rng.uniform(-1.5, 1.5, size=n), DT[dtype], offset)[0]
             for n in (1, 5, 4096, 20011, 0, 300)]
    want, factor = o.norm_and_factor([host(v) for v in views], size)
    got = ops["grad_norm"](grads=views, max_norm=size).cpu().numpy().astype(np.float64)
    # as in test_norm_matches
    assert abs(got[0] - want) <= 4.5 * o.U * want
    assert abs(got[1] - factor) <= 5.5 * o.U * factor


def test_norm_of_zeros_beside_tiny_and_ordinary_values(ops):
    zeros, tiny_ones = torch.zeros(100000, device="cuda"), torch.zeros(100000, device="cuda")
    zeros[::2] = -0.0
    assert ops["grad_norm"](grads=[zeros], max_norm=1.0).cpu().tolist() == [0.0, 1.0]
    tiny_ones[777] = 1e-30
    got = ops["grad_norm"](grads=[zeros, tiny_ones], max_norm=1.0).cpu().numpy()
    want = float(np.float32(1e-30))
    assert abs(float(got[0]) - want) <= 1.5 * o.U * want and got[1] == 1.0
    ordinary = torch.ones(100000, device="cuda")
    got = ops["grad_norm"](grads=[tiny_ones, ordinary], max_norm=1.0).cpu().numpy()
    want = 1e5 ** 0.5
    assert abs(float(got[0]) - want) <= 4.5 * o.U * want


def test_tensors_beyond_31_bits(ops):
    """A tensor of more than 2^31 elements beside a small one: the norm, and the step
    of its last elements."""
    n, tail = (1 << 31) + 70001, 80000
    g = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g[-tail:] = torch.randn(tail, device="cuda").to(torch.bfloat16)
    small = torch.randn(333, device="cuda").to(torch.bfloat16)
    want, _ = o.norm_and_factor([host(g[-tail:]), host(small)], 1.0)
    got = ops["grad_norm"](grads=[g, small], max_norm=1.0).cpu().numpy()
    assert abs(float(got[0]) - want) <= 4.5 * o.U * want
    p, m, v = (torch.zeros(n, device="cuda", dtype=d)
               for d in (torch.bfloat16, torch.float32, torch.float32))
    ops["adamw"](params=[p], grads=[g], exp_avg=[m], exp_avg_sq=[v], lr=1e-2, betas=(0.9, 0.95),
                 step=torch.zeros(1, dtype=torch.int64, device="cuda"))
    parts = [torch.zeros(tail, device="cuda", dtype=t.dtype) for t in (p, m, v)]
    ops["adamw"](params=parts[:1], grads=[g[-tail:].clone()], exp_avg=parts[1:2],
                 exp_avg_sq=parts[2:], lr=1e-2, betas=(0.9, 0.95),
                 step=torch.zeros(1, dtype=torch.int64, device="cuda"))
    for t, part in zip((p, m, v), parts):
        assert torch.equal(t[-tail:], part) and not t[:-tail].any()


def test_norm_is_the_same_every_time(ops):
    grads = [torch.randn(n, device="cuda", dtype=torch.bfloat16) for n in (1 << 21, 77, 1 << 19)]
    got = {tuple(ops["grad_norm"](grads=grads, max_norm=1.0).view(torch.int32).tolist())
           for _ in range(5)}
    assert len(got) == 1


# ---------------------------------------------------------------------------
# adamw

COMBOS = [("f32", "f32", False), ("f32", "bf16", False), ("f32", "f16", False),
          ("bf16", "bf16", False), ("bf16", "f32", True), ("bf16", "bf16", True),
          ("f16", "f16", True), ("f16", "f32", False), ("bf16", "f16", False),
          ("f16", "bf16", True)]


def half_eps(dtype):
    return torch.finfo(DT[dtype]).eps / 2 if dtype != "f32" else 0.0


def tiny(dtype):
    """Half the spacing of the type's smallest values."""
    return {"f32": 1e-45, "bf16": 1e-40, "f16": 2.0 ** -25}[dtype]


def step_lists(rng, sizes, param, grad, master, offset, first=False):
    z = 0.0 if first else 1.0
    lists = {"params": [guarded(rng.normal(size=n) * 0.05, DT[param], offset) for n in sizes],
             "grads": [guarded(rng.normal(size=n) * 10.0 ** rng.uniform(-4, 0), DT[grad], offset)
                       for n in sizes],
             "exp_avg": [guarded(z * rng.normal(size=n) * 1e-2, torch.float32, offset)
                         for n in sizes],
             "exp_avg_sq": [guarded(z * rng.normal(size=n) ** 2 * 1e-3, torch.float32, offset)
                            for n in sizes]}
    if master:
        lists["master"] = [guarded(rng.normal(size=n) * 0.05, torch.float32, offset)
                           for n in sizes]
    return lists


def check_adamw(ops, sizes, param, grad, master, offset=0, step=17, decay=0.1, scale=0.37,
                stream=None, lr=1e-2):
    rng = np.random.default_rng(len(sizes) * 1000 + sum(sizes) % 997 + offset)
    lists = step_lists(rng, sizes, param, grad, master, offset, first=step == 0)
    views = {k: [v for v, _ in ts] for k, ts in lists.items()}
    before = {k: [host(v) for v in ts] for k, ts in views.items()}
    count = torch.tensor([step], dtype=torch.int64, device="cuda")
    lr_t = torch.tensor([lr], device="cuda")
    scale_t = None if scale is None else torch.tensor([scale], device="cuda")
    decays = decay if isinstance(decay, list) else [decay] * len(sizes)
    torch.cuda.synchronize()
    got = ops["adamw"](step=count, lr=lr_t, betas=(HYPER["beta1"], HYPER["beta2"]),
                       eps=HYPER["eps"], weight_decay=decay, grad_scale=scale_t, stream=stream,
                       **views)
    torch.cuda.synchronize()
    assert got[0] is views["params"][0] and int(count) == step + 1
    s = 1.0 if scale is None else float(scale_t)
    for i in range(len(sizes)):
        old = before["master"][i] if master else before["params"][i]
        p, m, v, (bp, bm, bv) = o.adamw(
            old, before["grads"][i], before["exp_avg"][i], before["exp_avg_sq"][i], t=step + 1,
            lr=float(lr_t), decay=decays[i], scale=s, **HYPER)
        now = {k: host(ts[i]).astype(np.float64) for k, ts in views.items()}
        assert np.all(np.abs(now["exp_avg"] - m) <= bm)
        assert np.all(np.abs(now["exp_avg_sq"] - v) <= bv)
        if master:
            assert np.all(np.abs(now["master"] - p) <= bp)
            want = views["master"][i].to(DT[param])
            assert torch.equal(views["params"][i], want)
        else:
            slack = half_eps(param) * (np.abs(p) + bp) + tiny(param)
            assert np.all(np.abs(now["params"] - p) <= bp + slack)
        assert np.array_equal(now["grads"], before["grads"][i].astype(np.float64))
    assert all(untouched() for ts in lists.values() for _, untouched in ts)


@pytest.mark.parametrize("param,grad,master", COMBOS)
@pytest.mark.parametrize("offset", [0, 1])
def test_adamw_matches(ops, param, grad, master, offset):
    check_adamw(ops, [1, 2, 5, 255, 2048, 2049, 0, 70001], param, grad, master, offset)


@pytest.mark.parametrize("step", [0, 1, 100000])
@pytest.mark.parametrize("scale", [None, 1.0, 0.0])
def test_adamw_steps_and_scales(ops, step, scale):
    check_adamw(ops, [4099, 64], "f32", "f32", False, step=step, scale=scale)


def test_adamw_arrays_at_different_places(ops):
    """Arrays of one tensor that stand at different places mod 16 bytes."""
    rng = np.random.default_rng(5)
    n = 5003
    views = {k: guarded(np.abs(rng.normal(size=n)), torch.float32, off)
             for k, off in (("params", 1), ("grads", 2), ("exp_avg", 3), ("exp_avg_sq", 0))}
    before = {k: host(v) for k, (v, _) in views.items()}
    count = torch.zeros(1, dtype=torch.int64, device="cuda")
    ops["adamw"](step=count, lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.0,
                 **{k: [v] for k, (v, _) in views.items()})
    p, m, v, (bp, bm, bv) = o.adamw(before["params"], before["grads"], before["exp_avg"],
                                    before["exp_avg_sq"], t=1, lr=float(np.float32(1e-2)),
                                    decay=0.0, **HYPER)
    assert np.all(np.abs(host(views["params"][0]) - p) <= bp)
    assert np.all(np.abs(host(views["exp_avg"][0]) - m) <= bm)
    assert np.all(np.abs(host(views["exp_avg_sq"][0]) - v) <= bv)
    assert all(untouched() for _, untouched in views.values())


def test_adamw_of_a_long_list_with_a_decay_each(ops):
    rng = np.random.default_rng(6)
    sizes = [int(n) for n in rng.integers(0, 200, size=1100)]
    check_adamw(ops, sizes, "f32", "f32", False, decay=[0.01 * (i % 7) for i in range(1100)])


@pytest.mark.parametrize("name", ["adamw", "adamw8"])
@pytest.mark.parametrize("factor", [float("nan"), float("inf"), float("-inf")])
def test_a_factor_that_is_not_finite_skips_the_step(ops, name, factor):
    args = eight_state([300, 7], "f32", "f32", False, seed=1)[0] if name == "adamw8" else {
        k: [v for v, _ in ts] for k, ts in
        step_lists(np.random.default_rng(0), [300, 7], "f32", "f32", False, 0).items()}
    count = torch.tensor([5], dtype=torch.int64, device="cuda")
    before = {k: [t.clone() for t in ts] for k, ts in args.items() if k != "seed"}
    ops[name](step=count, lr=1e-2, betas=(0.9, 0.95), eps=1e-8,
              grad_scale=torch.tensor([factor], device="cuda"), **args)
    assert int(count) == 5
    for k, ts in before.items():
        for a, b in zip(ts, args[k]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), k


@pytest.mark.parametrize("eps", [1e-60, 1e-46, 1e-45, 1e-40])
@pytest.mark.parametrize("offset", [0, 1])
def test_adamw_eps_below_the_fp32_range(ops, eps, offset):
    """A value whose moments are zero does not move, however small eps is."""
    n = 1000
    views = {k: guarded(np.full(n, v), torch.float32, offset)[0]
             for k, v in (("params", 0.5), ("grads", 0.0), ("exp_avg", 0.0), ("exp_avg_sq", 0.0))}
    views["grads"][::3] = 1e-3
    ops["adamw"](step=torch.zeros(1, dtype=torch.int64, device="cuda"), lr=1e-2, eps=eps,
                 betas=(0.9, 0.95), weight_decay=0.0, **{k: [v] for k, v in views.items()})
    p, _, _, (bp, _, _) = o.adamw(
        np.full(n, 0.5), host(views["grads"]), np.zeros(n), np.zeros(n), t=1,
        lr=float(np.float32(1e-2)), beta1=0.9, beta2=0.95, eps=eps, decay=0.0)
    assert np.all(np.abs(host(views["params"]) - p) <= bp)
    assert np.all(host(views["params"])[1::3] == 0.5)


def test_a_binding_dropped_behind_its_launch(ops):
    """Inputs of another stream's pool stay as they are until the launch, which
    waits behind other work of its stream, has read them."""
    n, side = 1 << 22, torch.cuda.Stream()
    g = torch.ones(n, device="cuda")
    call, out = ops["grad_norm"].bind(grads=[g], max_norm=1.0, stream=side)
    call()   # loading a kernel waits for the device: not in what follows
    with torch.cuda.stream(side):
        torch.cuda._sleep(1)
    torch.cuda.synchronize()
    place = g.data_ptr()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)   # a tenth of a second
    call()
    del call, g
    other = [torch.full((n,), 5.0, device="cuda") for _ in range(4)]
    early = not side.query()
    torch.cuda.synchronize()
    assert early and float(out[0]) == n ** 0.5
    assert all(t.data_ptr() != place for t in other)


@pytest.mark.parametrize("betas", [(0.0, 0.0), (0.0, 0.95), (0.9, 0.0)])
def test_adamw_without_a_memory(ops, betas):
    """Betas of zero, with step, rate and factor of no dimensions."""
    rng = np.random.default_rng(3)
    views = {k: guarded(np.abs(rng.normal(size=777)), torch.float32, 1)[0]
             for k in ("params", "grads", "exp_avg", "exp_avg_sq")}
    old = {k: host(v) for k, v in views.items()}
    step = torch.zeros(1, dtype=torch.int64, device="cuda")[0]
    scale = ops["grad_norm"](grads=[views["grads"]], max_norm=1.0)[1]
    lr = torch.tensor(1e-2, device="cuda")
    ops["adamw"](step=step, lr=lr, betas=betas, eps=1e-8, weight_decay=0.1, grad_scale=scale,
                 **{k: [v] for k, v in views.items()})
    p, m, v, (bp, bm, bv) = o.adamw(old["params"], old["grads"], old["exp_avg"], old["exp_avg_sq"],
                                    t=1, lr=float(lr), beta1=betas[0], beta2=betas[1], eps=1e-8,
                                    decay=0.1, scale=float(scale))
    assert int(step) == 1
    assert np.all(np.abs(host(views["params"]) - p) <= bp)
    assert np.all(np.abs(host(views["exp_avg"]) - m) <= bm)
    assert np.all(np.abs(host(views["exp_avg_sq"]) - v) <= bv)


def test_adamw_of_two_types_with_a_step_each(ops):
    """A step of a model of two parameter types: two calls, one factor, a step tensor
    for each; the joint norm from the lists' norms."""
    rng = np.random.default_rng(4)
    kinds = [("bf16", "bf16", [300, 64]), ("f32", "f32", [33, 5])]
    lists = [{k: [v for v, _ in ts] for k, ts in step_lists(rng, n, p, g, False, 0).items()}
             for p, g, n in kinds]
    norms = [ops["grad_norm"](grads=li["grads"], max_norm=1.0) for li in lists]
    total = torch.hypot(norms[0][0], norms[1][0])
    factor = (0.1 / total).clamp(max=1.0)
    old = [{k: [host(t) for t in ts] for k, ts in li.items()} for li in lists]
    want, _ = o.norm_and_factor([g for li in old for g in li["grads"]], 1.0)
    assert abs(float(total) - want) <= 8 * o.U * want
    steps = [torch.full((1,), 6, dtype=torch.int64, device="cuda") for _ in lists]
    for li, step in zip(lists, steps):
        ops["adamw"](step=step, lr=1e-2, betas=(0.9, 0.95), grad_scale=factor, **li)
    for li, before, step, (kind, _, _) in zip(lists, old, steps, kinds):
        assert int(step) == 7
        for i, t in enumerate(li["params"]):
            p, _, _, (bp, _, _) = o.adamw(
                before["params"][i], before["grads"][i], before["exp_avg"][i],
                before["exp_avg_sq"][i], t=7, lr=float(np.float32(1e-2)), decay=0.0,
                scale=float(factor), **HYPER)
            slack = half_eps(kind) * (np.abs(p) + bp) + tiny(kind)
            assert np.all(np.abs(host(t) - p) <= bp + slack)


def test_adamw_on_a_side_stream(ops):
    check_adamw(ops, [70001, 3], "bf16", "bf16", True, stream=torch.cuda.Stream())


# ---------------------------------------------------------------------------
# adamw8


def eight_state(sizes, param, grad, master, offset=0, seed=11, first=False):
    rng = np.random.default_rng(sum(sizes) + offset + 31 * seed)
    blocks = [-(-n // o.BLOCK) for n in sizes]
    codes = lambda n, lo: torch.from_numpy(  # noqa: E731
        (rng.integers(lo, 121, size=n) * (not first)).astype(np.uint8))
    lists = {"params": [guarded(rng.normal(size=n) * 0.05, DT[param], offset) for n in sizes],
             "grads": [guarded(rng.normal(size=n) * 10.0 ** rng.uniform(-4, 0), DT[grad], offset)
                       for n in sizes]}
    if master:
        lists["master"] = [guarded(rng.normal(size=n) * 0.05, torch.float32, offset)
                           for n in sizes]
    for name, signed in (("exp_avg", True), ("exp_avg_sq", False)):
        lists[name] = []
        for n in sizes:
            c = codes(n, 0 if signed else 1)
            if signed:
                c = c | torch.from_numpy((rng.integers(0, 2, size=n) * 128).astype(np.uint8))
            view, ok = guarded(np.zeros(n), torch.float8_e4m3fn, offset)
            view.view(torch.uint8).copy_(c)
            lists[name].append((view, ok))
        lists[name + "_top"] = [guarded(np.exp(rng.uniform(-9, -3, size=b)) * (not first),
                                        torch.float32, offset) for b in blocks]
    args = {k: [v for v, _ in ts] for k, ts in lists.items()}
    args["seed"] = seed
    return args, [ok for ts in lists.values() for _, ok in ts]


def raw(t):
    return t.view(torch.uint8).cpu().numpy()


def check_adamw8(ops, sizes, param, grad, master, offset=0, step=17, seed=0x123456789ABCDEF,
                 scale=0.37, grads=None):
    args, guards = eight_state(sizes, param, grad, master, offset, seed, first=step == 0)
    if grads is not None:
        for t, g in zip(args["grads"], grads):
            t.copy_(torch.as_tensor(g))
    before = {k: [raw(t) if t.dtype == torch.float8_e4m3fn else host(t) for t in ts]
              for k, ts in args.items() if k != "seed"}
    count = torch.tensor([step], dtype=torch.int64, device="cuda")
    lr_t, scale_t = torch.tensor([1e-2], device="cuda"), torch.tensor([scale], device="cuda")
    ops["adamw8"](step=count, lr=lr_t, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1,
                  grad_scale=scale_t, **args)
    assert int(count) == step + 1
    key, block = o.step_key(seed, step + 1), 0
    for i, n in enumerate(sizes):
        m0 = o.opened(before["exp_avg"][i], before["exp_avg_top"][i])
        v0 = o.opened(before["exp_avg_sq"][i], before["exp_avg_sq_top"][i])
        m, v = o.moments32(m0, v0, before["grads"][i], beta1=0.9, beta2=0.95,
                           scale=float(scale_t))
        words = o.random_words(key, block, n)
        for x, name, half in ((m, "exp_avg", words & np.uint32(0xFFFF)),
                              (v, "exp_avg_sq", words >> np.uint32(16))):
            codes, tops = o.closed(x, half, name == "exp_avg_sq")
            assert np.array_equal(raw(args[name][i]), codes), (name, i)
            assert np.array_equal(host(args[name + "_top"][i]), tops), (name, i)
        old = before["master"][i] if master else before["params"][i]
        p, _, _, (bp, _, _) = o.adamw(old, before["grads"][i], m0, v0, t=step + 1,
                                      lr=float(lr_t), decay=0.1, scale=float(scale_t), **HYPER)
        now = host(args["params"][i]).astype(np.float64)
        if master:
            assert np.all(np.abs(host(args["master"][i]) - p) <= bp)
            assert torch.equal(args["params"][i], args["master"][i].to(DT[param]))
        else:
            assert np.all(np.abs(now - p) <= bp + half_eps(param) * (np.abs(p) + bp)
                          + tiny(param))
        block += -(-n // o.BLOCK)
    assert all(ok() for ok in guards)


@pytest.mark.parametrize("param,grad,master", COMBOS)
@pytest.mark.parametrize("offset", [0, 3])
def test_adamw8_matches_bit_for_bit(ops, param, grad, master, offset):
    check_adamw8(ops, [1, 7, 8, 255, 256, 257, 0, 2048, 2500, 30001], param, grad, master, offset)


@pytest.mark.parametrize("step", [0, 1, 1 << 33])
def test_adamw8_steps(ops, step):
    check_adamw8(ops, [1000, 40], "f32", "bf16", False, step=step)


@pytest.mark.parametrize("name,betas", [("adamw", (0.9, 0.999)), ("adamw8", (0.9, 0.95))])
def test_default_betas(ops, name, betas):
    """Those of the step's kind: 8-bit moments are not meant for a beta2 of 0.999."""
    def step(**more):
        args = eight_state([700], "f32", "f32", False, seed=5)[0] if name == "adamw8" else {
            k: [v for v, _ in ts] for k, ts in
            step_lists(np.random.default_rng(9), [700], "f32", "f32", False, 0).items()}
        ops[name](step=torch.zeros(1, dtype=torch.int64, device="cuda"), lr=1e-2, **args, **more)
        return [t.view(torch.uint8) for ts in args.values() if isinstance(ts, list) for t in ts]

    for a, b in zip(step(), step(betas=betas)):
        assert torch.equal(a, b)


def test_adamw8_of_a_long_list(ops):
    sizes = [int(n) for n in np.random.default_rng(8).integers(0, 600, size=800)]
    check_adamw8(ops, sizes, "bf16", "bf16", False)


def test_adamw8_blocks_of_zeros_and_of_tiny_values(ops):
    grads = [np.zeros(600, np.float32), np.full(600, 1e-18, np.float32)]
    grads[0][300] = 1e-16  # its second moment's block is below 2^-100
    check_adamw8(ops, [600, 600], "f32", "f32", False, step=0, scale=1.0, grads=grads)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_adamw8_block_that_is_not_finite(ops, bad):
    args, _ = eight_state([700], "f32", "f32", False)
    args["grads"][0][300] = bad
    count = torch.tensor([3], dtype=torch.int64, device="cuda")
    ops["adamw8"](step=count, lr=1e-2, betas=(0.9, 0.95), eps=1e-8, **args)
    for name in ("exp_avg", "exp_avg_sq"):
        top = host(args[name + "_top"][0])
        assert not np.isfinite(top[1]) and np.isfinite(top[[0, 2]]).all()
    # such a block reads back as not finite throughout, the others go on
    args["grads"][0][300] = 0.0
    ops["adamw8"](step=count, lr=1e-2, betas=(0.9, 0.95), eps=1e-8, **args)
    p = host(args["params"][0])
    assert np.isnan(p[256:512]).all() and np.isfinite(p[:256]).all()
    assert np.isfinite(p[512:]).all()


def test_adamw8_keeps_small_changes_on_average(ops):
    """A second moment that a step moves by less than a code's spacing still
    follows its formula on average: 64 steps of constant gradients, 2^16 values
    of one size, against the 64-bit recursion."""
    n, steps, beta2 = 1 << 16, 64, 0.95
    args = {"params": [torch.zeros(n, device="cuda")],
            "grads": [torch.full((n,), 1e-3, device="cuda")],
            "exp_avg": [torch.zeros(n, device="cuda").to(torch.float8_e4m3fn)],
            "exp_avg_sq": [torch.zeros(n, device="cuda").to(torch.float8_e4m3fn)],
            "exp_avg_top": [torch.zeros(n // 256, device="cuda")],
            "exp_avg_sq_top": [torch.zeros(n // 256, device="cuda")], "seed": 3}
    # one large value a block sets the top, so that the others fall between codes
    args["grads"][0][::256] = 0.05
    count = torch.zeros(1, dtype=torch.int64, device="cuda")
    for _ in range(steps):
        ops["adamw8"](step=count, lr=1e-3, betas=(0.9, beta2), eps=1e-8, **args)
    v = o.opened(raw(args["exp_avg_sq"][0]), host(args["exp_avg_sq_top"][0])).astype(np.float64)
    small = np.ones(n, bool)
    small[::256] = False
    want = (1 - beta2 ** steps) * 1e-6
    # one value's deviation is at most a third of it (a spacing of at most the whole
    # value near the smallest codes, over the square root of a memory of ten steps);
    # the mean of 65280 has one 255 times smaller, and 6 of these are 0.8%
    assert abs(v[small].mean() / want - 1) < 0.01


# ---------------------------------------------------------------------------
# what is refused, before anything runs


def test_refusals(ops):
    t = lambda n=4, d=torch.float32: torch.zeros(n, device="cuda", dtype=d)  # noqa: E731
    with pytest.raises(ValueError):
        ops["grad_norm"](grads=[t()], max_norm=0.0)
    with pytest.raises(ValueError):
        ops["grad_norm"](grads=[], max_norm=1.0)
    with pytest.raises(TypeError):
        ops["grad_norm"](grads=[t(), t(4, torch.bfloat16)], max_norm=1.0)
    with pytest.raises(TypeError):
        ops["grad_norm"](grads=[torch.zeros(4, 4, device="cuda").t()[1:]], max_norm=1.0)
    with pytest.raises(TypeError):
        ops["grad_norm"](grads=[t(4, torch.float64)], max_norm=1.0)
    with pytest.raises(TypeError):
        ops["grad_norm"](grads=[torch.zeros(4)], max_norm=1.0)
    with pytest.raises(ValueError):
        g = t(8)
        ops["grad_norm"](grads=[g], max_norm=1.0, out=g[:2])
    good = dict(params=[t()], grads=[t()], exp_avg=[t()], exp_avg_sq=[t()],
                step=t(1, torch.int64), lr=1e-3)
    same = t()
    for change, error in [(dict(grads=[t(5)]), ValueError), (dict(grads=[]), ValueError),
                          (dict(exp_avg=[t(4, torch.bfloat16)]), TypeError),
                          (dict(step=t(1)), TypeError), (dict(step=t(2, torch.int64)), ValueError),
                          (dict(betas=(1.0, 0.9)), ValueError), (dict(eps=-1.0), ValueError),
                          (dict(master=[t()]), ValueError), (dict(weight_decay=[0.1, 0.1]),
                                                             ValueError),
                          (dict(lr=t(2)), ValueError), (dict(grad_scale=t(2)), ValueError),
                          (dict(params=[same], exp_avg=[same]), ValueError),
                          (dict(grads=[same], params=[same]), ValueError)]:
        with pytest.raises(error):
            ops["adamw"](**{**good, **change})
    twice = {k: v * 2 for k, v in good.items() if isinstance(v, list)}
    with pytest.raises(ValueError):
        ops["adamw"](**{**good, **twice})
    f8 = torch.float8_e4m3fn
    eight = dict(params=[t()], grads=[t()], exp_avg=[t(4).to(f8)], exp_avg_sq=[t(4).to(f8)],
                 exp_avg_top=[t(1)], exp_avg_sq_top=[t(1)], step=t(1, torch.int64), lr=1e-3,
                 seed=1)
    for change, error in [(dict(exp_avg=[t()]), TypeError), (dict(exp_avg_top=[t(2)]), ValueError),
                          (dict(eps=0.0), ValueError), (dict(seed=-1), ValueError),
                          (dict(seed=None), ValueError)]:
        with pytest.raises(error):
            ops["adamw8"](**{**eight, **change})


def test_numbers_that_are_not_finite_or_beyond_fp32_are_refused(ops):
    """Before anything runs, as ValueError: the C entries take floats."""
    t = lambda n=4, d=torch.float32: torch.zeros(n, device="cuda", dtype=d)  # noqa: E731
    for bad in (1e-50, float("nan"), -1.0):
        with pytest.raises(ValueError):
            ops["grad_norm"](grads=[t()], max_norm=bad)
    assert ops["grad_norm"](grads=[t()], max_norm=1e39).cpu().tolist() == [0.0, 1.0]
    good = dict(params=[t()], grads=[t()], exp_avg=[t()], exp_avg_sq=[t()],
                step=t(1, torch.int64), lr=1e-3)
    for change in (dict(weight_decay=float("nan")), dict(weight_decay=[float("inf")]),
                   dict(eps=float("inf")), dict(eps=float("nan")),
                   dict(betas=(0.9, float("nan")))):
        with pytest.raises(ValueError):
            ops["adamw"](**{**good, **change})
    assert int(good["step"]) == 0


def test_gradients_may_be_given_twice(ops):
    """What is only read may overlap: one gradient for two tensors."""
    g = torch.randn(100, device="cuda")
    p = [torch.ones(100, device="cuda") for _ in range(2)]
    z = [torch.zeros(100, device="cuda") for _ in range(4)]
    ops["adamw"](params=p, grads=[g, g], exp_avg=z[:2], exp_avg_sq=z[2:],
                 step=torch.zeros(1, dtype=torch.int64, device="cuda"), lr=1e-3)
    assert torch.equal(p[0], p[1])
