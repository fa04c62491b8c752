"""The Vx declarations of the library's ops (vx_amd/vx/packages/vx_nn/lib.vx)
against the C header: the same functions with the same types in the same
order, and wrappers that call them by their parameters."""

import re
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
LIB = re.sub(r"//[^\n]*", "", (ROOT / "vx_amd/vx/packages/vx_nn/lib.vx").read_text())
HEADER = re.sub(r"/\*.*?\*/", "", (ROOT / "include/vx_hip_ops.h").read_text(), flags=re.S)

C_TYPES = {"int8_t": "i8", "uint16_t": "bf16", "float": "f32", "int32_t": "i32", "int64_t": "i64", "void": "i8",
           "vx_llama_sampling": "i8"}


def split(args: str) -> list[str]:
    """At the commas that are in no bracket."""
    parts, depth = [""], 0
    for c in args:
        depth += (c in "([<") - (c in ")]>")
        if c == "," and depth == 0:
            parts.append("")
        else:
            parts[-1] += c
    return [" ".join(a.split()) for a in parts if a.strip()]


def in_c() -> dict[str, list[str]]:
    """Name -> each parameter as "name : type" with its pointer's kind."""
    out = {}
    for m in re.finditer(r"\b(vx_\w+)\s*\(([^()]*)\)\s*;", HEADER):
        params = []
        for p in split(m.group(2)):
            q = re.fullmatch(r"(const\s+)?(\w+)\s*(\*?)\s*(\w+)", p)
            if q and q.group(2) in C_TYPES:
                kind = "" if not q.group(3) else "*const " if q.group(1) else "*mut "
                params.append(f"{q.group(4)} : {kind}{C_TYPES[q.group(2)]}")
            else:
                params.append(p)
        out[m.group(1)] = params
    return out


def in_vx() -> dict[str, list[str]]:
    block = LIB[LIB.index('extern "C" {'):]
    block = block[:block.index("\n}")]
    return {m.group(1): [re.sub(r"\s+in Memory::M", "", p) for p in split(m.group(2))]
            for m in re.finditer(r"fn (vx_\w+)(?:<[^>]*>)?\(([^()]*)\)", block)}


OPS = ["vx_nn_flash_attention_fwd_bf16", "vx_nn_gemv_i8_bf16", "vx_nn_rope_append_bf16", "vx_nn_rope_append_f32",
       "vx_nn_flash_attention_shared_bf16", "vx_nn_flash_attention_shared_workspace", "vx_nn_sample_f32",
       "vx_nn_sample_bf16", "vx_nn_sample_workspace", "vx_llama_i8_sample"]


@pytest.mark.parametrize("op", OPS)
def test_declared_as_in_the_header(op):
    assert in_vx()[op] == in_c()[op]


def test_every_op_is_declared():
    assert {n for n in in_c() if n.startswith("vx_nn_")} == {n for n in in_vx() if n.startswith("vx_nn_")}


WRAPPERS = ["flash_attention_causal", "gemv_i8", "rope_append", "flash_attention_shared", "sample", "sample_bf16"]


@pytest.mark.parametrize("name", WRAPPERS)
def test_wrappers_pass_what_the_op_takes(name):
    """As many arguments as the op has, pointers of operands of its element
    types, read where it reads and written where it writes."""
    m = re.search(rf"\nfn {name}<M : Memory>\((.*?)\) -> i32 \{{\s*return unsafe \{{\s*(vx_\w+)\((.*?)\)\s*\}};\s*\}}", LIB,
                  re.S)
    params = {}
    for p in split(m.group(1)):
        who, kind = (x.strip() for x in p.split(":", 1))
        t = re.match(r"(&mut |&)Tensor<(\w+), \[(.*?)\]", kind)
        params[who] = (t.group(1) == "&mut ", t.group(2), t.group(3).count("?")) if t else kind
    args, want = split(m.group(3)), in_c()[m.group(2)]
    assert len(args) == len(want)
    used = set()
    for a, w in zip(args, want):
        kind = w.split(" : ")[1]
        p = re.fullmatch(r"(\w+)\.as_(mut_)?ptr\(\)", a)
        d = re.fullmatch(r"(\w+)\.dim\((\d)\) as i64", a)
        if kind.startswith("*"):
            assert p, (a, w)
            assert params[p.group(1)][:2] == (kind.startswith("*mut"), kind.split()[1]), (a, w)
            assert bool(p.group(2)) == kind.startswith("*mut"), (a, w)
            # an operand goes to the parameter of its name
            assert p.group(1) == w.split(" : ")[0], (a, w)
            used.add(p.group(1))
        elif d:
            assert kind == "i64" and int(d.group(2)) < params[d.group(1)][2], (a, w)
        elif a in params:
            assert params[a] == kind and a == w.split(" : ")[0], (a, w)
            used.add(a)
        else:
            assert a == "1" and w == "causal : i32", (a, w)
    assert used == set(params)
