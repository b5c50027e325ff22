"""The training-step operator package: ``lib<package>.so`` or ``.a``, its
header, manifest and report, in the layout of a compiled package
(``artifact.py``).

Its operators are hand-written (``csrc/b200_train_*.cu``) and take what the
entry language cannot say: lists of tensors, 16-bit and 8-bit element types,
states updated in place, rows.  The C interface is
``include/loom/b200_train.h``; ``loom_b200.train_ops.TrainPackage`` loads it.
"""

from __future__ import annotations

import json
import os
import shlex
import shutil
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path
from typing import List, Tuple

from .artifact import (CSRC, CUDA_ARCH, GENCODE, BuildError, PackageResult, _run, _write)

PACKAGE = "b200_train"
HEADER = Path(__file__).resolve().parent.parent / "include" / "loom" / f"{PACKAGE}.h"
SOURCES = ("b200_train_lists.cu", "b200_train_norms.cu", "b200_train_rows.cu")

# the element types of block_norm's residual stream and branch
ROW_TYPES = (("float", "float"), ("float", "__nv_bfloat16"), ("float", "__half"),
             ("__nv_bfloat16", "__nv_bfloat16"), ("__half", "__half"))


def _units() -> List[Tuple[str, str, List[str]]]:
    """(source, object, defines) of every compilation."""
    units = [(s, s[:-3] + ".o", []) for s in SOURCES[:2]]
    for x, b in ROW_TYPES:
        for backward in (0, 1):
            obj = f"rows_{x.strip('_')}_{b.strip('_')}_{'backward' if backward else 'forward'}.o"
            units.append((SOURCES[2], obj, [f"-DLOOM_ROWS_X={x}", f"-DLOOM_ROWS_B={b}",
                                            f"-DLOOM_ROWS_BACKWARD={backward}"]))
    return units

# entry name -> (what it does, whether it takes a workspace)
ENTRIES = {
    "grad_norm": ("2-norm of a list of tensors and its clipping factor", True),
    "adamw": ("AdamW step over a list of tensors, fp32 states", True),
    "adamw8": ("AdamW step over a list of tensors, 8-bit states", True),
    "block_norm": ("norms after and before a block with its gate and residual scale", False),
    "block_norm_backward": ("gradients of block_norm", True),
}


def symbol_of(entry: str) -> str:
    return f"loom_train_{entry}"


def _commands(nvcc: str, include_dir: str, out_dir: str, artifact: str, kind: str):
    """(compile commands, link commands); the sources compile side by side."""
    base = [nvcc, "-std=c++17", "-O3", "-gencode", GENCODE, "-fmad=false", "-lineinfo",
            "-Xptxas", "-O3", f"-I{include_dir}", f"-I{CSRC}", "-c", "-Xcompiler", "-fPIC"]
    compiles, objects = [], []
    for name, obj, defines in _units():
        obj = os.path.join(out_dir, "src-gen", obj)
        compiles.append(base + defines + ["-o", obj, str(CSRC / name)])
        objects.append(obj)
    if kind == "shared":
        return compiles, [[nvcc, "-shared", "-gencode", GENCODE, "-o", artifact] + objects]
    return compiles, [["ar", "rcs", artifact] + objects]


def _entry_json(entry: str) -> dict:
    text, workspace = ENTRIES[entry]
    sym = symbol_of(entry)
    d = {"entry_name": entry, "module_name": "train", "symbol_name": sym,
         "stream_symbol": sym + "_stream", "packed_symbol": sym + "_packed",
         "description": text}
    if workspace:
        d["workspace_symbol"] = sym + "_workspace_size"
    return d


def generate_train_package(out_dir: str, kind: str = "shared", nvcc: str = "nvcc",
                           build: bool = True) -> PackageResult:
    """Build the operator package into `out_dir`."""
    if kind not in ("shared", "static"):
        raise BuildError(f"unknown artifact kind {kind} (expected shared or static)")
    out_dir = os.path.abspath(out_dir)
    include_root = os.path.join(out_dir, "include")
    header = os.path.join(include_root, "loom", f"{PACKAGE}.h")
    artifact = os.path.join(out_dir, f"lib{PACKAGE}.{'so' if kind == 'shared' else 'a'}")
    _write(header, HEADER.read_text(encoding="utf-8"))
    compiles, links = _commands(nvcc, include_root, out_dir, artifact, kind)
    if build:
        if shutil.which(nvcc) is None and not os.path.exists(nvcc):
            raise BuildError("nvcc is required on PATH for the Loom B200 backend")
        os.makedirs(os.path.join(out_dir, "src-gen"), exist_ok=True)
        with ThreadPoolExecutor(os.cpu_count() or 1) as pool:
            list(pool.map(_run, compiles))
        if kind == "static" and os.path.exists(artifact):
            os.remove(artifact)
        for cmd in links:
            _run(cmd)
    commands: List[str] = [shlex.join(c) for c in compiles + links]
    sources = [str(CSRC / name) for name in SOURCES]
    manifest = os.path.join(out_dir, "manifest.json")
    report = os.path.join(out_dir, "report.md")
    _write(manifest, json.dumps({
        "mode": "operators", "target_backend": "cuda", "backend": "loom-b200",
        "package_name": PACKAGE, "artifact_kind": kind, "cuda_arch": CUDA_ARCH,
        "artifact_path": artifact, "header_path": header, "source_path": sources,
        "entries": [_entry_json(e) for e in ENTRIES], "build_commands": commands}, indent=2))
    lines = ["# Loom Operator Package Report", "", f"- package: `{PACKAGE}`",
             f"- artifact kind: `{kind}`", f"- CUDA arch: `{CUDA_ARCH}`",
             f"- artifact: `{artifact}`", f"- header: `{header}`", ""]
    for e, (text, workspace) in ENTRIES.items():
        lines += [f"## `{symbol_of(e)}`", "", f"- operator: `{e}`: {text}",
                  f"- workspace function: `{symbol_of(e)}_workspace_size`" if workspace
                  else "- workspace: none", ""]
    lines += ["## Build Commands", ""] + [f"- `{c}`" for c in commands] + [""]
    _write(report, "\n".join(lines))
    return PackageResult(str(CSRC), PACKAGE, artifact, header, sources[0], manifest, report,
                         commands)
