"""The 64-bit restatements of the training-step operators against themselves:
gradients against differences, the random words' distribution, and the 8-bit
codes against torch's own float8_e4m3fn."""

import numpy as np
import pytest
import torch

from oracle import train_oracle as o


@pytest.mark.parametrize("forms", ["all", "no gate", "one gate", "two gates", "no post", "no pre",
                                   "no h"])
def test_gradients_against_differences(forms):
    rng = np.random.default_rng(7)
    rows, width = 4, 5
    runs = {"one gate": 1, "two gates": 2, "no gate": 0}.get(forms, rows)
    has_h = forms != "no h"
    inputs = {"x": rng.normal(size=(rows, width))}
    if has_h:
        inputs["h"] = rng.normal(size=(rows, width))
        if runs:
            inputs["gate"] = rng.normal(size=(runs, width))
        if forms != "no post":
            inputs["post"] = rng.normal(size=width)
    if forms != "no pre":
        inputs["pre"] = rng.normal(size=width)
    cy, cz = rng.normal(size=(rows, width)), rng.normal(size=(rows, width))
    kw = dict(offset=0.5, a=0.7, b=1.3) if has_h else dict(offset=0.5)
    flags = dict(post_norm=has_h and forms != "no post", pre_norm=forms != "no pre", eps=1e-3)

    def value(inp):
        y, z, *_ = o.block_norm(inp["x"], inp.get("h"), inp.get("gate"), inp.get("post"),
                                inp.get("pre"), **flags, **kw)
        return float((cy * y).sum() + ((cz * z).sum() if z is not None else 0.0))

    y, z, q, r, _ = o.block_norm(inputs["x"], inputs.get("h"), inputs.get("gate"),
                                 inputs.get("post"), inputs.get("pre"), **flags, **kw)
    grads = o.block_norm_grads(y, inputs.get("h"), inputs.get("gate"), inputs.get("post"),
                               inputs.get("pre"), q, r, cy, cz if z is not None else None, **kw)
    names = {"x": "dx", "h": "dh", "gate": "dgate", "post": "dpost_weight", "pre": "dpre_weight"}
    step = 1e-5
    for key, a in inputs.items():
        got, _ = grads[names[key]]
        for at in np.ndindex(a.shape):
            up, down = ({k: x.copy() for k, x in inputs.items()} for _ in range(2))
            up[key][at] += step
            down[key][at] -= step
            slope = (value(up) - value(down)) / (2 * step)
            # central differences: a third derivative of order 10 times step^2, and
            # rounding of values of order 10 over the step
            assert abs(slope - got[at]) < 1e-7, (key, at, slope, got[at])


def test_without_h_the_residual_scale_has_no_part():
    """y is x then, whatever the scale: its gradient too."""
    rng = np.random.default_rng(17)
    x, cy, cz = (rng.normal(size=(3, 6)) for _ in range(3))
    pre = rng.normal(size=6)
    kw = dict(offset=0.5, a=0.5)

    def value(x):
        y, z, *_ = o.block_norm(x, None, None, None, pre, eps=1e-3, **kw)
        return float((cy * y).sum() + (cz * z).sum())

    y, _, q, r, _ = o.block_norm(x, None, None, None, pre, eps=1e-3, **kw)
    assert q is None and np.array_equal(y, x)
    got, _ = o.block_norm_grads(y, None, None, None, pre, q, r, cy, cz, **kw)["dx"]
    step = 1e-5
    for at in np.ndindex(x.shape):
        up, down = x.copy(), x.copy()
        up[at] += step
        down[at] -= step
        # as above: a third derivative of order 10 times step^2, rounding over the step
        assert abs((value(up) - value(down)) / (2 * step) - got[at]) < 1e-7, at


def test_e4m3_values_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    ours = o.e4m3_values()
    theirs = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(theirs[:127], ours[:127]) and np.isnan(theirs[127])
    assert np.array_equal(theirs[128:255], -ours[:127])


def test_rounding_is_to_a_neighbour_and_even_on_average():
    rng = np.random.default_rng(3)
    x = np.zeros(4096, dtype=np.float32)
    x[:] = np.exp(rng.uniform(-18, 0, x.size)) * rng.choice([-1, 1], x.size)
    x[0] = 1.0
    words = [o.random_words(o.step_key(99, t), 0, x.size) for t in range(1, 401)]
    grid = o.e4m3_values()[:127]
    total = np.zeros(x.size)
    for w in words:
        codes, tops = o.closed(x, w & np.uint32(0xFFFF), False)
        got = o.opened(codes, tops).astype(np.float64)
        a = np.abs(x.astype(np.float64)) * o.TOP / np.repeat(tops, o.BLOCK).astype(np.float64)
        low = np.searchsorted(grid, a * (1 + 1e-6), side="right") - 1
        unit = np.repeat(tops, o.BLOCK).astype(np.float64) / o.TOP
        down = np.searchsorted(grid, a * (1 - 1e-6), side="right") - 1
        near = np.abs(got) / unit
        assert np.all((near >= grid[down] * (1 - 1e-6))
                      & (near <= grid[np.minimum(low + 1, 126)] * (1 + 1e-6)))
        assert np.all((got == 0) | (np.sign(got) == np.sign(x)))
        total += got
    spacing = np.maximum(np.abs(x) / 8, np.repeat(tops, o.BLOCK) * 2.0 ** -17)
    # the mean of 400 draws of a two-point distribution within one spacing has a
    # deviation of at most 1/40 of it; 4096 values stay within 6 of these
    assert np.all(np.abs(total / 400 - x) < 6 / 40 * spacing)


def test_random_words_are_even_and_independent():
    n = 1 << 18
    a = o.random_words(o.step_key(5, 1), 0, n)
    b = o.random_words(o.step_key(5, 2), 0, n)
    unit = lambda w, s: ((w >> np.uint32(s)) & np.uint32(0xFFFF)) / 65536 - 0.5  # noqa: E731
    rows = [unit(a[j::8], s) for j in range(8) for s in (0, 16)]
    rows += [unit(b[j::8], s) for j in range(2) for s in (0, 16)]
    c = np.corrcoef(rows)
    np.fill_diagonal(c, 0)
    # correlations of 2^15 independent pairs have a deviation of 2^-7.5; 380 pairs
    # stay within 4.5 of these
    assert np.abs(c).max() < 4.5 * 2.0 ** -7.5
    for r in rows:
        assert abs(r.mean()) < 5 * 12 ** -0.5 * 2.0 ** -7.5
    # words of consecutive tensors differ: the blocks are counted through the list
    assert not np.array_equal(a[256:512], o.random_words(o.step_key(5, 1), 0, 256))
    assert np.array_equal(a[256:512], o.random_words(o.step_key(5, 1), 1, 256))
