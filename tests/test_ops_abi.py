"""The operators' C ABI on the CPU: exports and argument blocks match the header, and entries refuse before any GPU call."""

import ctypes
import re
import subprocess

import pytest

from conftest import ROOT

STRUCTS = {"emmy_ops_norm_args": "NormArgs", "emmy_ops_rotary_args": "RotaryArgs",
           "emmy_ops_cache4_append_args": "Cache4AppendArgs", "emmy_ops_cache4_attend_args": "Cache4AttendArgs",
           "emmy_ops_blockfp8_quantize_args": "BlockFp8QuantizeArgs", "emmy_ops_blockfp8_args": "BlockFp8Args",
           "emmy_ops_blockfp8_linear_args": "BlockFp8LinearArgs"}


def test_exports_match_header():
    import emmyrt
    header = (ROOT / "include" / "emmyrt_ops.h").read_text()
    declared = set(re.findall(r"\b(emmy_ops_\w+)\s*\(", header))
    assert declared == set(emmyrt.OPS_SIGNATURES)
    for name in declared:
        assert hasattr(emmyrt.ops_lib(), name)


def c_name(field: str, struct: str) -> str:
    if struct == "emmy_ops_blockfp8_linear_args":
        own = {"x": "x", "x_stride": "x_stride", "x_dtype": "x_dtype", "reserved2": "reserved"}
        return own.get(field, "product." + field)
    if field.startswith("cache_"):
        return "cache." + field[6:]
    if struct == "emmy_ops_rotary_args" and field[-1] in "01":
        return f"{field[:-1]}[{field[-1]}]"
    return field


def test_argument_blocks_match_header(tmp_path):
    import emmyrt
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "emmyrt_ops.h"', "int main(void) {"]
    want = []
    for c, py in STRUCTS.items():
        block = getattr(emmyrt, py)
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        want.append(ctypes.sizeof(block))
        for name, _ in block._fields_:
            if not name.startswith("_"):
                lines.append(f'printf("%zu\\n", offsetof({c}, {c_name(name, c)}));')
                want.append(getattr(block, name).offset)
    src = tmp_path / "t.c"
    src.write_text("\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "t")], check=True)
    got = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == want


def refused(entry, args, what):
    import emmyrt
    lib = emmyrt.ops_lib()
    assert getattr(lib, entry)(ctypes.byref(args) if args is not None else None, 0, 0) == -3
    assert what in lib.emmy_ops_last_error().decode()


def norm(**change):
    import emmyrt
    a = dict(x=1 << 20, block=2 << 20, y=3 << 20, h=4 << 20, x_stride=64, block_stride=64, y_stride=64, h_stride=64,
             rows=4, dim=64, rows_per_gate=4)
    return emmyrt.NormArgs(**{**a, **change})


@pytest.mark.parametrize("change,what", [
    (dict(dtype=3), "element type"), (dict(dim=0), "dim"), (dict(dim=16385), "dim"), (dict(rows=-1), "rows"),
    (dict(kind=2), "kind"), (dict(x=0), "needed"), (dict(x=(1 << 20) + 1), "aligned"), (dict(y_stride=63), "overlap"),
    (dict(gate=5 << 20, rows_per_gate=0), "rows_per_gate"), (dict(gate=5 << 20, gate_dtype=9), "element type"),
    (dict(post_norm=1, post_weight=(5 << 20) + 2), "aligned")])
def test_norm_refusals(change, what):
    refused("emmy_ops_residual_norm", norm(**change), what)


def rotary(**change):
    import emmyrt
    a = dict(x0=1 << 20, out0=2 << 20, x_token0=64, x_head0=64, out_token0=64, out_head0=64, heads0=1, positions=3 << 20,
             turns=4 << 20, tokens=4, dim=64, rotary=64, magnitude=1.0)
    return emmyrt.RotaryArgs(**{**a, **change})


@pytest.mark.parametrize("change,what", [
    (dict(dtype=-1), "element type"), (dict(rotary=63), "rotary"), (dict(rotary=0), "rotary"), (dict(rotary=66), "rotary"),
    (dict(layout=2), "layout"), (dict(tokens=-1), "tokens"), (dict(heads0=-1), "heads"), (dict(heads1=1 << 20), "heads"),
    (dict(positions=0), "positions"), (dict(positions=(3 << 20) + 4, positions_64=1), "positions"), (dict(out0=0), "needed"),
    (dict(heads1=1), "needed"), (dict(x0=(1 << 20) + 2), "aligned")])
def test_rotary_refusals(change, what):
    refused("emmy_ops_rotary", rotary(**change), what)


def append(**change):
    import emmyrt
    a = dict(cache_k=1 << 20, cache_v=2 << 20, cache_k_meta=3 << 20, cache_v_meta=4 << 20, cache_pages=4, cache_heads=2,
             cache_page=16, cache_dim=64, k=5 << 20, v=6 << 20, slots=7 << 20, k_token=128, k_head=64, v_token=128,
             v_head=64, tokens=4)
    return emmyrt.Cache4AppendArgs(**{**a, **change})


@pytest.mark.parametrize("change,what", [
    (dict(cache_dim=96), "head dim"), (dict(cache_heads=0), "cache of"), (dict(cache_page=0), "cache of"),
    (dict(cache_pages=-1), "cache of"), (dict(cache_k=0), "no memory"), (dict(cache_v=(2 << 20) + 8), "16 bytes"),
    (dict(cache_k_meta=(3 << 20) + 2), "on 4"), (dict(dtype=7), "element type"), (dict(tokens=-2), "tokens"),
    (dict(k=0), "needed"), (dict(slots=(7 << 20) + 4, slots_64=1), "aligned"), (dict(k_stored=8), "16 bytes"),
    (dict(tokens=0x7fffffff, cache_heads=4096), "too many")])
def test_append_refusals(change, what):
    refused("emmy_ops_cache4_append", append(**change), what)


def attend(**change):
    import emmyrt
    a = dict(cache_k=1 << 20, cache_v=2 << 20, cache_k_meta=3 << 20, cache_v_meta=4 << 20, cache_pages=4, cache_heads=2,
             cache_page=16, cache_dim=64, q=5 << 20, out=6 << 20, table=7 << 20, lengths=8 << 20, workspace=9 << 20,
             workspace_bytes=1 << 40, q_batch=256, q_token=256, q_head=64, out_batch=256, out_token=256, out_head=64,
             table_stride=2, batch=3, tokens=1, q_heads=4, max_pages=2, dtype=2, scale=1.0)
    return emmyrt.Cache4AttendArgs(**{**a, **change})


@pytest.mark.parametrize("change,what", [
    (dict(cache_dim=32), "head dim"), (dict(dtype=0), "f16 or bf16"), (dict(batch=-1), "batch"), (dict(batch=4097), "batch"),
    (dict(tokens=-1), "tokens"), (dict(q_heads=0), "heads"), (dict(q_heads=3), "heads"), (dict(tokens=1 << 20, q_heads=8), "tokens"),
    (dict(max_pages=-1), "pages"), (dict(max_pages=1 << 30), "pages"), (dict(q=0), "needed"), (dict(table=0), "needed"),
    (dict(workspace=0), "workspace"), (dict(workspace=(9 << 20) + 8), "workspace"), (dict(q=(5 << 20) + 1), "aligned"),
    (dict(lengths=(8 << 20) + 2), "aligned"), (dict(batch=4096, cache_heads=4096, q_heads=4096, max_pages=1 << 20), "too many")])
def test_attend_refusals(change, what):
    refused("emmy_ops_cache4_attend", attend(**change), what)


def test_attend_workspace_of_an_unknown_dim():
    import emmyrt
    n = ctypes.c_uint64()
    assert emmyrt.ops_lib().emmy_ops_cache4_attend_workspace(96, 0, ctypes.byref(n)) == -3
    assert emmyrt.ops_lib().emmy_ops_cache4_attend_workspace(64, 0, None) == -3


def product(**change):
    import emmyrt
    a = dict(xq=1 << 20, xs=2 << 20, wq=3 << 20, ws=4 << 20, y=5 << 20, status=6 << 20, xq_stride=144, xs_stride=8, wq_stride=144,
             ws_stride=2, y_stride=10, m=8, n=10, k=130, dtype=2)
    return emmyrt.BlockFp8Args(**{**a, **change})


@pytest.mark.parametrize("change,what", [
    (dict(dtype=4), "element type"), (dict(n=0), "n 0"), (dict(m=-1), "xq"), (dict(k=0), "xq"), (dict(xq=0), "xq"),
    (dict(xq=(1 << 20) + 8), "xq"), (dict(xq_stride=136), "xq"), (dict(xq_stride=128), "xq"), (dict(k=143, wq_stride=160, xq_stride=128), "xq"),
    (dict(wq_stride=136), "wq"), (dict(wq=(3 << 20) + 1), "wq"), (dict(xs=0), "xs"), (dict(xs_stride=7), "xs"), (dict(xs_stride=10), "xs"),
    (dict(ws_stride=1, n=300, y_stride=300), "overlap"), (dict(y_stride=9), "overlap"), (dict(y=(5 << 20) + 1), "y"), (dict(status=0), "status"),
    (dict(parts=(7 << 20) + 4, parts_bytes=64), "parts"), (dict(m=0x7fffff00, n=0x7fffff00, y_stride=0x7fffff00, xs_stride=0x7fffff00), "y of")])
def test_product_refusals(change, what):
    refused("emmy_ops_blockfp8_product", product(**change), what)


def quantise(**change):
    import emmyrt
    a = dict(x=1 << 20, q=2 << 20, s=3 << 20, x_stride=130, q_stride=144, s_stride=8, rows=8, cols=130, dtype=2)
    return emmyrt.BlockFp8QuantizeArgs(**{**a, **change})


@pytest.mark.parametrize("change,what", [
    (dict(dtype=5), "element type"), (dict(rows=-1), "x of"), (dict(cols=0), "x of"), (dict(x=0), "x is needed"),
    (dict(x=(1 << 20) + 1), "x is needed"), (dict(q=(2 << 20) + 4), "q is needed"), (dict(q_stride=130), "16"), (dict(q_stride=128), "overlap"),
    (dict(s=2), "s is needed"), (dict(s_stride=7), "overlap"), (dict(square=1, rows=300, s_stride=1), "overlap")])
def test_quantise_refusals(change, what):
    refused("emmy_ops_blockfp8_quantize", quantise(**change), what)


@pytest.mark.parametrize("change,what", [(dict(x=0), "x is needed"), (dict(x_dtype=7), "element type"), (dict(x_stride=100), "overlap"),
                                         (dict(x_stride=100, m=2), "overlap"), (dict(wq=0), "wq")])
def test_linear_refusals(change, what):
    import emmyrt
    a = {n: getattr(product(), n) for n, _ in emmyrt.BlockFp8Args._fields_}
    refused("emmy_ops_blockfp8_linear", emmyrt.BlockFp8LinearArgs(**{**a, "x": 8 << 20, "x_stride": 130, "x_dtype": 2, **change}), what)


@pytest.mark.parametrize("entry", ["emmy_ops_residual_norm", "emmy_ops_rotary", "emmy_ops_cache4_append", "emmy_ops_cache4_attend",
                                   "emmy_ops_blockfp8_quantize", "emmy_ops_blockfp8_product", "emmy_ops_blockfp8_linear"])
def test_no_arguments(entry):
    refused(entry, None, "no arguments")
