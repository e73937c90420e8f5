"""Writes the listing of the Python layer's public names (``python -m rocshmem_b200.utils.gen_pydoc docs/PYTHON_API.md``):
for every module the public functions and classes with their signatures and the first paragraph of their
docstrings. The C++ / CUDA API has its own listing (``gen_api``)."""
from __future__ import annotations

import importlib
import inspect
import sys
from typing import List

MODULES = ["rocshmem_b200.runtime", "rocshmem_b200.ops.collectives", "rocshmem_b200.ops.moe", "rocshmem_b200.ops.moe_host",
           "rocshmem_b200.ops.gemm", "rocshmem_b200.ops.attention", "rocshmem_b200.ops.host_algorithms", "rocshmem_b200.models.moe_ffn",
           "rocshmem_b200.models.tp_mlp", "rocshmem_b200.parallel.layout", "rocshmem_b200.parallel.pipeline",
           "rocshmem_b200.parallel.membership", "rocshmem_b200.parallel.elastic", "rocshmem_b200.parallel.data_parallel", "rocshmem_b200.parallel.ulysses", "rocshmem_b200.parallel.ring",
           "rocshmem_b200.parallel.context", "rocshmem_b200.utils.checkpoint", "rocshmem_b200.utils.trace",
           "rocshmem_b200.utils.roofline", "rocshmem_b200.baselines.nccl_collectives", "rocshmem_b200.baselines.tp_mlp",
           "rocshmem_b200.baselines.moe", "rocshmem_b200.baselines.ep"]


def _first_paragraph(obj) -> str:
    doc = inspect.getdoc(obj) or ""
    return " ".join(doc.split("\n\n")[0].split())


def _signature(obj) -> str:
    try:
        return str(inspect.signature(obj))
    except (TypeError, ValueError):
        return "(...)"


def _public(mod):
    for name, obj in vars(mod).items():
        if name.startswith("_") or getattr(obj, "__module__", None) != mod.__name__:
            continue
        if inspect.isfunction(obj) or inspect.isclass(obj):
            yield name, obj


def markdown() -> str:
    out: List[str] = ["# Python API listing", "",
                      "Generated by `python -m rocshmem_b200.utils.gen_pydoc docs/PYTHON_API.md` from the docstrings.", ""]
    for modname in MODULES:
        mod = importlib.import_module(modname)
        out += [f"## `{modname}`", "", _first_paragraph(mod), ""]
        for name, obj in _public(mod):
            if inspect.isclass(obj):
                out.append(f"* **class `{name}{_signature(obj)}`** — {_first_paragraph(obj)}")
                for mname, meth in vars(obj).items():
                    if mname.startswith("_") or not (inspect.isfunction(meth) or isinstance(meth, property)):
                        continue
                    if isinstance(meth, property):
                        out.append(f"  * `{mname}` (property) — {_first_paragraph(meth.fget)}")
                    else:
                        out.append(f"  * `{mname}{_signature(meth)}` — {_first_paragraph(meth)}")
            else:
                out.append(f"* `{name}{_signature(obj)}` — {_first_paragraph(obj)}")
        out.append("")
    return "\n".join(out)


def main(argv=None) -> int:
    import argparse
    ap = argparse.ArgumentParser(description="Lists every public Python name of the package with its signature and "
                                             "the first paragraph of its docstring, as Markdown.")
    ap.add_argument("file", nargs="?", help="write here instead of standard output")
    args = ap.parse_args(argv)
    text = markdown()
    if args.file:
        with open(args.file, "w") as f:
            f.write(text)
    else:
        sys.stdout.write(text)
    return 0


if __name__ == "__main__":
    sys.exit(main())
