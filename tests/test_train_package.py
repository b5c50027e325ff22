"""The training-step operator package: its files, its header from plain C, and
what its C entries refuse (checked before any CUDA call, so without a GPU)."""

import ctypes
import json
import os
import re
import shutil
import subprocess
import sys

import pytest

from loom_b200 import train_ops, train_package
from loom_b200.build import TRAIN_DIR, build_train, load_train

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SRC = os.path.join(HERE, "c", "train_smoke.c")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")
OK, INVALID, SMALL = 0, 1, 2
FAKE = 0x10000          # an aligned address that is never dereferenced on the host


@pytest.fixture(scope="module")
def ops():
    if not os.path.exists(os.path.join(TRAIN_DIR, "libb200_train.so")):
        if shutil.which("nvcc") is None:
            pytest.skip("needs nvcc")
        build_train()
    return load_train()


@pytest.fixture(scope="module")
def static_package(tmp_path_factory):
    if shutil.which("nvcc") is None:
        pytest.skip("needs nvcc")
    out = tmp_path_factory.mktemp("train_static")
    proc = subprocess.run([sys.executable, "-m", "loom_b200", "train-ops", "--out", str(out),
                           "--kind", "static"], cwd=ROOT, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr
    assert proc.stdout.strip() == str(out / "libb200_train.a")
    return out


def test_package_files(static_package):
    manifest = json.loads((static_package / "manifest.json").read_text())
    assert manifest["package_name"] == "b200_train" and manifest["artifact_kind"] == "static"
    assert [e["entry_name"] for e in manifest["entries"]] == list(train_package.ENTRIES)
    header = (static_package / "include" / "loom" / "b200_train.h").read_text()
    assert header == (train_package.HEADER).read_text()
    report = (static_package / "report.md").read_text()
    for e in manifest["entries"]:
        assert e["symbol_name"] in report


def test_header_declares_what_the_library_exports(ops):
    text = re.sub(r"/\*.*?\*/", "", train_package.HEADER.read_text(), flags=re.S)
    declared = set(re.findall(r"\b(loom_train_\w+)\(", text))
    listed = set()
    for e in ops.manifest["entries"]:
        listed |= {e["symbol_name"], e["stream_symbol"], e["packed_symbol"]}
        if "workspace_symbol" in e:
            listed.add(e["workspace_symbol"])
    assert declared == listed
    for name in declared:
        assert getattr(ops.lib, name) is not None
    # the loader's argument counts are the header's, and its structures have the
    # header's fields' types in the header's order
    ctype = {"int64_t": ctypes.c_int64, "int": ctypes.c_int, "float": ctypes.c_float,
             "double": ctypes.c_double, "size_t": ctypes.c_size_t, "uint64_t": ctypes.c_uint64}
    for e in ops.manifest["entries"]:
        body = re.search(r"typedef struct %s_args \{(.*?)\}" % e["symbol_name"], text, re.S)
        fields = [f.strip() for f in body.group(1).split(";") if f.strip()]
        kinds = [ctypes.c_void_p if "*" in f else ctype[f.split()[0]] for f in fields]
        assert kinds == [t for _, t in train_ops._PACKED[e["entry_name"]]._fields_]
    for e in ops.manifest["entries"]:
        sig = re.search(re.escape(e["symbol_name"]) + r"\(([^)]*)\);", text).group(1)
        assert len(sig.split(",")) == len(train_ops._ARGTYPES[e["entry_name"]])


@pytest.fixture(scope="module")
def c_programs(ops, static_package, tmp_path_factory):
    if shutil.which("gcc") is None or shutil.which("nvcc") is None:
        pytest.skip("needs gcc and nvcc")
    out = tmp_path_factory.mktemp("train_c")
    shared, static = str(out / "shared"), str(out / "static")
    for cmd in (["gcc", "-std=c11", "-O2", "-Wall", "-Werror", f"-I{ROOT}/include",
                 f"-I{CUDA}/include", SRC, "-o", shared, f"-L{TRAIN_DIR}", "-lb200_train",
                 f"-Wl,-rpath,{TRAIN_DIR}", f"-L{CUDA}/lib64", "-lcudart", "-lm"],
                ["nvcc", "-O2", f"-I{static_package}/include", SRC, "-o", static,
                 str(static_package / "libb200_train.a"), "-lm"]):
        proc = subprocess.run(cmd, capture_output=True, text=True)
        assert proc.returncode == 0, proc.stderr
    return shared, static


def test_c_programs_build(c_programs):
    assert all(os.path.exists(p) for p in c_programs)


@pytest.mark.gpu
def test_c_programs_run(c_programs):
    for path in c_programs:
        proc = subprocess.run([path], capture_output=True, text=True, timeout=120)
        assert proc.returncode == 0, proc.stderr
        assert "train_smoke ok" in proc.stdout


def test_row_plans(tmp_path):
    """Host arithmetic only: no kernel of the program is launched."""
    if shutil.which("nvcc") is None:
        pytest.skip("needs nvcc")
    program = str(tmp_path / "row_plan_check")
    proc = subprocess.run(["nvcc", "-std=c++17", "-O1", "-gencode", train_package.GENCODE,
                           f"-I{train_package.CSRC}", os.path.join(HERE, "c", "row_plan_check.cu"),
                           "-o", program], capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr
    proc = subprocess.run([program], capture_output=True, text=True, timeout=120)
    assert proc.returncode == 0 and "row plans ok" in proc.stdout, proc.stderr


def test_every_gradient_kernel_can_be_chosen(ops):
    """Rows of the widest CTA come one group a thread through stages, and so do rows
    with a gate row per run: the library holds no others with two groups."""
    if shutil.which("nm") is None:
        pytest.skip("needs nm")
    text = subprocess.run(["nm", "-C", ops.path], capture_output=True, text=True).stdout
    forms = set(re.findall(r"block_norm_grad_kernel<[^,]*, [^,]*, (\w+), \w+, (\d), \w+, (\d+), "
                           r"\(loomb::Gate\)(\d)", text))
    assert {("true", "1", "1024", "2"), ("true", "2", "512", "1")} <= forms
    assert not any(groups == "2" and (threads == "1024" or gate == "2")
                   for _, groups, threads, gate in forms)


def test_dependent_kernels_promise_no_read_only_data():
    """A kernel that waits for the grid before it is resident while that grid still
    writes.  A const __restrict__ pointer promises that nobody does, and allows
    loads through a path that the wait says nothing about."""
    seen = 0
    for path in sorted(train_package.CSRC.glob("*.cuh")):
        parts = re.split(r"(?=__global__)", path.read_text())[1:]
        for part in parts:
            kernel = part[:part.index("\n}")]
            if "wait_for_prerequisite_grid()" not in kernel:
                continue
            seen += 1
            assert not re.search(r"const[\w:<>\s]*\*\s*(const\s+)?__restrict__", kernel), (
                path.name, kernel[:200])
    assert seen >= 11


# ---------------------------------------------------------------------------
# refusals of the C entries


def _ptrs(*values):
    return (ctypes.c_void_p * len(values))(*values)


def _i64(*values):
    return (ctypes.c_int64 * len(values))(*values)


def _call(op, stream, **args):
    """The stream form with these arguments in the declared order, and the packed
    form, which has to say the same."""
    values = [ctypes.addressof(v) if isinstance(v, ctypes.Array) else v for v in args.values()]
    status = op.stream_fn(*values, stream)
    packed = train_ops._PACKED[op.name](*values)
    assert op.packed_fn(ctypes.addressof(packed), stream) == status
    assert op.packed_fn(None, stream) == INVALID
    return status


def norm_args(**change):
    a = dict(count=2, grads=_ptrs(FAKE, FAKE), sizes=_i64(4, 5), dtype=0, max_norm=1.0, out=FAKE,
             ws=FAKE, ws_size=1 << 20)
    a.update(change)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(count=-1), INVALID), (dict(grads=None), INVALID), (dict(sizes=None), INVALID),
    (dict(sizes=_i64(4, -1)), INVALID), (dict(grads=_ptrs(FAKE, 0)), INVALID),
    (dict(grads=_ptrs(FAKE, FAKE + 2)), INVALID), (dict(dtype=3), INVALID),
    (dict(dtype=-1), INVALID), (dict(max_norm=0.0), INVALID), (dict(max_norm=-1.0), INVALID),
    (dict(max_norm=float("nan")), INVALID), (dict(out=None), INVALID),
    (dict(out=FAKE + 2), INVALID), (dict(ws=None), SMALL), (dict(ws_size=0), SMALL),
    (dict(sizes=_i64(4, (1 << 40) + 1)), INVALID)], ids=str)
def test_norm_refuses(ops, change, status):
    assert _call(ops["grad_norm"], None, **norm_args(**change)) == status


def adam_args(eight, **change):
    a = dict(count=2, params=_ptrs(FAKE, FAKE), grads=_ptrs(FAKE, FAKE), m=_ptrs(FAKE, FAKE),
             v=_ptrs(FAKE, FAKE))
    if eight:
        a.update(m_top=_ptrs(FAKE, FAKE), v_top=_ptrs(FAKE, FAKE))
    a.update(master=None, sizes=_i64(4, 5), decay=(ctypes.c_double * 2)(0.1, 0.0), param=0, grad=0,
             lr=FAKE, beta1=0.9, beta2=0.95, eps=1e-8, scale=None, step=FAKE)
    if eight:
        a["seed"] = 1
    a.update(ws=FAKE, ws_size=1 << 20)
    a.update(change)
    return a


ADAM_BAD = [
    (dict(count=-1), INVALID), (dict(params=None), INVALID), (dict(grads=_ptrs(0, FAKE)), INVALID),
    (dict(m=None), INVALID), (dict(v=_ptrs(FAKE, 0)), INVALID), (dict(sizes=_i64(-1, 5)), INVALID),
    (dict(decay=None), INVALID), (dict(decay=(ctypes.c_double * 2)(0.1, float("nan"))), INVALID),
    (dict(param=3), INVALID), (dict(grad=-1), INVALID), (dict(lr=None), INVALID),
    (dict(lr=FAKE + 1), INVALID), (dict(beta1=1.0), INVALID), (dict(beta2=-0.1), INVALID),
    (dict(beta2=float("nan")), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=float("inf")), INVALID), (dict(step=None), INVALID), (dict(step=FAKE + 4), INVALID),
    (dict(scale=FAKE + 2), INVALID), (dict(master=_ptrs(FAKE, FAKE)), INVALID),
    (dict(params=_ptrs(FAKE + 2, FAKE)), INVALID),
    (dict(param=1, master=_ptrs(FAKE, FAKE + 2)), INVALID),
    (dict(param=1, params=_ptrs(FAKE + 1, FAKE)), INVALID),
    (dict(ws=None), SMALL), (dict(ws_size=100), SMALL)]


@pytest.mark.parametrize("change,status", ADAM_BAD, ids=str)
def test_adamw_refuses(ops, change, status):
    assert _call(ops["adamw"], None, **adam_args(False, **change)) == status


@pytest.mark.parametrize("change,status", ADAM_BAD + [
    (dict(m_top=None), INVALID), (dict(v_top=_ptrs(FAKE, FAKE + 2)), INVALID),
    (dict(eps=0.0), INVALID), (dict(eps=1e-60), INVALID), (dict(eps=1e-40), INVALID)], ids=str)
def test_adamw8_refuses(ops, change, status):
    assert _call(ops["adamw8"], None, **adam_args(True, **change)) == status


@pytest.mark.parametrize("sizes", [(1 << 40, 1), (1 << 40, 1 << 40), (1 << 39, (1 << 39) + 1),
                                   ((1 << 62), (1 << 62)), (5, (1 << 63) - 1)], ids=str)
@pytest.mark.parametrize("name", ["grad_norm", "adamw", "adamw8"])
def test_lists_beyond_their_most_values_are_refused_before_a_launch(ops, name, sizes):
    """A step that had begun would have counted: the whole list is looked at first."""
    args = norm_args() if name == "grad_norm" else adam_args(name == "adamw8")
    args["sizes"] = _i64(*sizes)
    assert _call(ops[name], None, **args) == INVALID


def rows_args(**change):
    a = dict(x=FAKE, x_stride=64, h=FAKE, h_stride=64, gate=FAKE, gate_stride=64, gate_rows=2,
             post=FAKE, pre=FAKE, rows=4, width=64, x_type=1, h_type=1, post_norm=1, pre_norm=1,
             eps=1e-6, offset=0.0, a=1.0, b=1.0, y=FAKE, z=FAKE, post_rstd=None, pre_rstd=None)
    a.update(change)
    return a


ROWS_BAD = [
    (dict(rows=-1), INVALID), (dict(rows=1 << 31), INVALID), (dict(width=0), INVALID),
    (dict(width=32769), INVALID), (dict(width=(1 << 32) + 64), INVALID),
    (dict(x_type=1, h_type=0), INVALID), (dict(x_type=1, h_type=2), INVALID),
    (dict(x_type=5), INVALID), (dict(post_norm=2), INVALID), (dict(pre_norm=-1), INVALID),
    (dict(h=None), INVALID), (dict(post_norm=0), INVALID), (dict(pre_norm=0), INVALID),
    (dict(gate_rows=3), INVALID), (dict(gate_rows=0), INVALID), (dict(gate_rows=-2), INVALID),
    (dict(offset=float("nan")), INVALID), (dict(a=float("inf")), INVALID),
    (dict(b=float("nan")), INVALID), (dict(x_stride=-64), INVALID), (dict(x=FAKE + 1), INVALID),
    (dict(h_stride=1 << 31), INVALID),
    (dict(gate=FAKE + 1), INVALID), (dict(post=FAKE + 1), INVALID)]


@pytest.mark.parametrize("change,status", ROWS_BAD + [
    (dict(x=None), INVALID), (dict(y=None), INVALID), (dict(z=None), INVALID),
    (dict(z=FAKE + 1), INVALID), (dict(pre_rstd=FAKE + 2), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=float("nan")), INVALID), (dict(rows=0, h=None, x=None, y=None, z=None), OK)], ids=str)
def test_block_norm_refuses(ops, change, status):
    assert _call(ops["block_norm"], None, **rows_args(**change)) == status


def grad_args(**change):
    a = dict(y=FAKE, x_stride=64, h=FAKE, h_stride=64, gate=FAKE, gate_stride=64, gate_rows=2,
             post=FAKE, pre=FAKE, post_rstd=FAKE, pre_rstd=FAKE, dy=FAKE, dy_stride=64, dz=FAKE,
             dz_stride=64, rows=4, width=64, x_type=1, h_type=1, post_norm=1, pre_norm=1,
             offset=0.0, a=1.0, b=1.0, dx=FAKE, dh=FAKE, dgate=FAKE, dpost=FAKE, dpre=FAKE,
             ws=FAKE, ws_size=1 << 30)
    if "x" in change:
        change = {("y" if k == "x" else k): v for k, v in change.items()}
    a.update(change)
    return a


@pytest.mark.parametrize("change,status", ROWS_BAD + [
    (dict(y=None), INVALID), (dict(dz=None), INVALID), (dict(pre_rstd=None), INVALID),
    (dict(post_rstd=None), INVALID), (dict(dx=None), INVALID), (dict(dh=None), INVALID),
    (dict(dgate=None), INVALID), (dict(gate=None), INVALID), (dict(post=None), INVALID),
    (dict(pre=None), INVALID), (dict(dy=FAKE + 1), INVALID), (dict(dz_stride=-1), INVALID),
    (dict(ws=None), SMALL), (dict(ws_size=1000), SMALL)], ids=str)
def test_block_norm_backward_refuses(ops, change, status):
    assert _call(ops["block_norm_backward"], None, **grad_args(**change)) == status


def test_workspace_sizes(ops):
    assert ops["grad_norm"].workspace_size(-1) == 0
    assert ops["grad_norm"].workspace_size(0) > 0
    assert ops["grad_norm"].workspace_size(5000) > ops["grad_norm"].workspace_size(5)
    assert ops["adamw"].workspace_size(-1) == 0 and ops["adamw8"].workspace_size(3) > 0
    size = ops["block_norm_backward"].workspace_size
    assert size(-1, 64, 0) == 0 and size(5, 0, 0) == 0
    assert size(4096, 64, 2) >= size(4096, 64, 0) > 0
    assert ops["block_norm"].workspace_size() == 0


def test_given_outputs_that_overlap_are_refused():
    import torch
    buf = torch.zeros(4, 32)
    a, b, c = buf[0], buf[1], buf[1:3]
    train_ops._rows_disjoint("op", [a, None, buf[:0]], [b, c, None])
    for written, read in (([a, a], []), ([a, None, a], []), ([b, c], []), ([c, b], []),
                          ([a], [a]), ([b], [a, c]), ([buf[:, 8:], a[:9]], [])):
        with pytest.raises(ValueError):
            train_ops._rows_disjoint("op", written, read)


def test_host_tensors_are_refused(ops):
    import torch
    t = torch.zeros(4)
    for name, args in (("grad_norm", dict(grads=[t], max_norm=1.0)), ("block_norm", dict(x=t))):
        with pytest.raises(TypeError):
            ops[name](**args)
        with pytest.raises(TypeError):
            ops[name].bind(**args)
    with pytest.raises(ValueError):
        ops["grad_norm"](grads=[], max_norm=1.0)
