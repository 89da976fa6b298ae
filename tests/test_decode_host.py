"""Host side of decoding in 4 bits and of beam search (no GPU needed: every case is rejected before any device call): the C
header's declarations and layouts, refusals of the wrappers (ValueError) and of the C ABI (a status with a message)."""
import ctypes as C
import hashlib
import math
import os
import re
import subprocess

import pytest
import torch

import decode_reference as R
from utttcompanion_amd import _native as N
from utttcompanion_amd import build
from utttcompanion_amd import kernels as K

STRUCTS = {"uttt_linear4_args": N.Linear4Args, "uttt_readout4_args": N.Readout4Args, "uttt_swa_tree4_args": N.SwaTree4Args,
           "uttt_kv_commit4_args": N.KvCommit4Args, "uttt_kv_values4_args": N.KvValues4Args,
           "uttt_kv_fork4_args": N.KvFork4Args, "uttt_beam_select_args": N.BeamSelectArgs}


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(build.LIB_PATH):
        build.build()
    return N.load_library()


def test_every_declared_symbol_is_exported_and_typed(lib):
    text = re.sub(r"/\*.*?\*/", "", open(N.DECODE_HEADER_PATH).read(), flags=re.S)
    names = set(re.findall(r"\b(uttt_[a-z0-9_]+)\s*\(", text))
    assert names == set(N.DECODE_SIGNATURES)
    assert all(hasattr(lib, name) for name in names)
    assert lib.uttt_decode_abi_version() == N.DECODE_ABI_VERSION


def test_declarations_belong_to_the_abi_version():
    """Other declarations take another UTTT_DECODE_ABI_VERSION: the digest changes together with it."""
    text = re.sub(r"/\*.*?\*/", " ", open(N.DECODE_HEADER_PATH).read(), flags=re.S)
    text = " ".join(re.sub(r"#define UTTT_DECODE_ABI_VERSION \d+", "", text).split())
    assert (N.DECODE_ABI_VERSION, hashlib.sha256(text.encode()).hexdigest()[:16]) == (1, "b849dd2f076add7d")


def test_library_without_these_entry_points_is_refused(tmp_path, monkeypatch):
    (tmp_path / "old.c").write_text(f"int uttt_abi_version(void) {{ return {N.ABI_VERSION}; }}\n"
                                    f"int uttt_serve_abi_version(void) {{ return {N.SERVE_ABI_VERSION}; }}\n")
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(tmp_path / "old.so"), str(tmp_path / "old.c")], check=True)
    monkeypatch.setattr(N, "_lib", None)
    with pytest.raises(RuntimeError, match="decoding ABI version 0, expected"):
        N.load_library(str(tmp_path / "old.so"))


def test_struct_layouts_match_the_c_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{N.DECODE_HEADER_PATH}"', 'int main(void) {']
    for cname, py in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {field} %zu\\n", offsetof({cname}, {field}));' for field, _ in py._fields_]
    lines.append("return 0; }")
    (tmp_path / "layout.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, stdout=subprocess.PIPE, text=True).stdout
    got = {tuple(line.split()[:2]): int(line.split()[2]) for line in out.splitlines()}
    for cname, py in STRUCTS.items():
        assert got.pop((cname, "size")) == C.sizeof(py), cname
        for field, _ in py._fields_:
            assert got.pop((cname, field)) == getattr(py, field).offset, f"{cname}.{field}"
    assert not got


# ---------------------------------------------------------------------------- the wrappers
def refused(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def asks(t):
    return t.clone().requires_grad_()


def test_packing_needs_no_gpu():
    w = torch.randn(20, 70)
    p = K.pack_weight4(w)
    padded = torch.zeros(20, 96)
    padded[:, :70] = w
    assert p.data.shape == (2, 1, 1152) and torch.equal(R.weight_values(p.data, 20, 70), R.values(*R.fours(padded))[:, :70])
    both = K.pack_weight4(torch.stack([w, -w]))
    assert torch.equal(both.data[0], p.data) and both.data.shape == (2, 2, 1, 1152) and both[1:] == (20, 70)
    for bad in (torch.zeros(3), torch.zeros(0, 4), torch.zeros(2, 2, 2, 2), torch.zeros(3, 4, dtype=torch.int32)):
        refused("floating", K.pack_weight4, bad)


def test_linear_refusals():
    p, x = K.pack_weight4(torch.ones(8, 40)), torch.zeros(3, 40)
    refused("no CPU path", K.linear4, x, p)
    refused(r"x must be \(m, 40\)", K.linear4, x[:, 1:], p)
    refused(r"x must be \(m, 40\)", K.linear4, x[0], p)
    refused("float32 or bfloat16", K.linear4, x.half(), p)
    refused("packed weight of", K.linear4, x, K.Weight4(p.data, 17, 40))
    refused("packed weight of", K.linear4, x, K.Weight4(p.data.int(), 8, 40))
    refused("one matrix", K.linear4, x, K.Weight4(p.data[None], 8, 40))
    refused("lie together", K.linear4, x, K.Weight4(torch.zeros(1, 1, 1160, dtype=torch.uint8)[..., 8:], 8, 40))
    for eps in (-1.0, math.nan, math.inf):
        refused("x_eps", K.linear4, x, p, x_eps=eps)


def test_readout_refusals():
    up, down = K.pack_weight4(torch.ones(2, 128, 64)), K.pack_weight4(torch.ones(2, 64, 128))
    x, ln = torch.zeros(2, 1, 64), torch.ones(64)
    refused("no CPU path", K.readout4, x, up, up, down, ln, ln)
    refused(r"\(B, T, D\)", K.readout4, x[0], up, up, down, ln, ln)
    refused("multiples of 64", K.readout4, torch.zeros(2, 1, 65), up, up, down, ln, ln)
    refused("w_down must be a packed", K.readout4, x, up, up, up, ln, ln)
    refused("one matrix or 3", K.readout4, torch.zeros(3, 1, 64), up, up, down, ln, ln)
    refused("ln_bias", K.readout4, x, up, up, down, ln, ln[1:])
    refused("norm weight", K.readout4, x, up, up, down, ln, ln, x_norm=(ln[1:], 1e-6))
    for eps in (0.0, -1.0, math.nan):
        refused("eps must be", K.readout4, x, up, up, down, ln, ln, eps)
        refused("eps must be", K.readout4, x, up, up, down, ln, ln, x_norm=(ln, eps))


def cache_and_nodes(n=2, t=3, hkv=1, hd=64, window=40, sinks=2):
    c = K.kv_cache4(n, hkv, window=window, sinks=sinks, head_dim=hd, device=torch.device("cpu"))
    return c, torch.zeros(n, t, hkv, hd), torch.zeros(n, dtype=torch.int64)


def test_cache_refusals():
    c, k, pos = cache_and_nodes()
    assert c.shape == (2, 1, 3, 2304)
    refused("head_dim must be", K.kv_cache4, 2, 1, window=4, sinks=0, head_dim=96, device="cpu")
    refused("head_dim must be", K.kv_cache4, 2, 1, window=0, sinks=0, head_dim=64, device="cpu")
    ids, counts = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    refused("no CPU path", K.kv_commit4, k, k, ids, counts, c, pos, 40, 2)
    refused("blocks of", K.kv_commit4, k, k, ids, counts, c, pos, 70, 2)
    refused("blocks of", K.kv_commit4, k, k, ids, counts, c, pos, 40, 33)
    refused("window must be", K.kv_commit4, k, k, ids, counts, c, pos, 0, 2)
    refused("uint8", K.kv_commit4, k, k, ids, counts, c.int(), pos, 40, 2)
    refused("one row per cache", K.kv_commit4, k, k[:, 1:], ids, counts, c, pos, 40, 2)
    refused("share one dtype", K.kv_commit4, k, k.bfloat16(), ids, counts, c, pos, 40, 2)
    refused("float32 or bfloat16", K.kv_commit4, k.half(), k.half(), ids, counts, c, pos, 40, 2)
    refused("nodes must be int32", K.kv_commit4, k, k, ids.long(), counts, c, pos, 40, 2)
    refused("counts must be", K.kv_commit4, k, k, ids, counts.long(), c, pos, 40, 2)
    refused("positions must be", K.kv_commit4, k, k, ids, counts, c, pos.int(), 40, 2)
    refused("lie together", K.kv_values4, torch.zeros(2, 2, 6, 2304, dtype=torch.uint8)[:, :, ::2], 40, 2)
    refused("16-byte aligned", K.kv_values4, torch.zeros(c.numel() + 8, dtype=torch.uint8)[8:].view(c.shape), 40, 2)
    refused("no CPU path", K.kv_values4, c, 40, 2)
    refused("float32 or bfloat16", K.kv_values4, c, 40, 2, torch.float16)
    refused("no CPU path", K.kv_fork4, c, counts, pos, 40, 2)
    refused("sources must be", K.kv_fork4, c, counts.long(), pos, 40, 2)
    many = K.kv_cache4(129, 1, window=1, sinks=0, head_dim=64, device=torch.device("cpu"))
    refused("at most 128", K.kv_fork4, many, torch.zeros(129, dtype=torch.int32), None, 1)


def test_tree_refusals():
    c, k, pos = cache_and_nodes()
    q = torch.zeros(2, 3, 4, 64)
    call = lambda **kw: K.swa_tree4(kw.pop("q", q), kw.pop("k", k), kw.pop("v", k), kw.pop("c", c), kw.pop("pos", pos),  # noqa: E731
                                    kw.pop("window", 40), sinks=kw.pop("sinks", 2), **kw)
    refused("no CPU path", call)
    refused("q must be", call, q=q[0])
    refused("1 to 64 nodes", call, q=torch.zeros(2, 65, 4, 64))
    refused("new keys", call, q=torch.zeros(2, 2, 4, 64))
    refused("new keys", call, q=torch.zeros(2, 3, 4, 128))
    refused("multiple of n_kv_heads", call, c=c.repeat(1, 3, 1, 1), k=k.repeat(1, 1, 3, 1), v=k.repeat(1, 1, 3, 1))
    refused("share one dtype", call, v=k.bfloat16())
    refused("blocks of", call, window=100)
    refused("positions", call, pos=pos.int())
    refused("counts", call, counts=pos)
    refused("parents", call, parents=torch.zeros(2, 3))
    tab = torch.zeros(10, 64)
    refused("both be given", call, cos=tab)
    refused("tables", call, cos=tab, sin=tab[:, 1:])
    refused("tables", call, cos=tab.double(), sin=tab.double())


def test_beam_refusals():
    x, s = torch.zeros(6, 100), torch.zeros(6)
    refused("no CPU path", K.beam_select, x, s, 3)
    refused("divide the rows", K.beam_select, x, s, 4)
    refused("1 to 32", K.beam_select, x, s, 0)
    refused("1 to 32", K.beam_select, torch.zeros(33, 9), torch.zeros(33), 33)
    refused("logits must be", K.beam_select, x[0], s, 3)
    refused("logits must be", K.beam_select, x.t(), s, 3)
    refused("scores must be", K.beam_select, x, s.double(), 3)
    refused("scores must be", K.beam_select, x, s[1:], 3)
    refused("ended must be", K.beam_select, x, s, 3, ended=s)
    refused("at most 8", K.beam_select, x, s, 3, banned=range(9))
    refused("excluded ids", K.beam_select, x, s, 3, banned=(-1,))
    refused("pad", K.beam_select, x, s, 3, pad=100)
    refused("pad", K.beam_select, x, s, 3, pad=-1)
    refused("active_limit", K.beam_select, x, s, 3, active_limit=-2)
    refused("float32 or bfloat16", K.beam_select, x.half(), s, 3)
    refused("2\\^20", K.beam_select, torch.zeros(1, (1 << 20) + 1), s[:1], 1)


def test_operands_that_ask_for_gradients_are_refused():
    """Under no_grad they pass on."""
    p, x = K.pack_weight4(torch.ones(64, 64)), torch.zeros(2, 64)
    c, k, pos = cache_and_nodes()
    ln = torch.ones(64)
    calls = [lambda: K.linear4(asks(x), p), lambda: K.linear4(x, p, residual=asks(x)),
             lambda: K.readout4(asks(x)[None], p, p, p, ln, ln), lambda: K.readout4(x[None], p, p, p, asks(ln), ln),
             lambda: K.swa_tree4(asks(k), k, k, c, pos, 40, sinks=2), lambda: K.swa_tree4(k, asks(k), k, c, pos, 40, sinks=2),
             lambda: K.kv_commit4(k, asks(k), None, None, c, pos, 40, 2),
             lambda: K.beam_select(asks(x), torch.zeros(2), 2), lambda: K.beam_select(x, asks(torch.zeros(2)), 2)]
    for call in calls:
        with pytest.raises(ValueError, match="forward-only"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="no CPU path"):
            call()


# ---------------------------------------------------------------------------- the C ABI
def test_c_refusals(lib):
    """Before any launch, each with its message."""
    def refused_c(fn, a, match):
        assert fn(C.byref(a), None) == 1 and match in lib.uttt_last_error().decode(), lib.uttt_last_error()

    for name in ("uttt_linear4", "uttt_readout4", "uttt_swa_tree4", "uttt_kv_commit4", "uttt_kv_values4", "uttt_kv_fork4",
                 "uttt_beam_select"):
        assert getattr(lib, name)(None, None) == 1 and b"args is NULL" in lib.uttt_last_error()
    a = N.Linear4Args(m=2, n=8, k=40, act_dtype=1, x=16, x_row_stride=40, w=32, out=64, out_row_stride=8)
    for field, value, match in (("act_dtype", 2, "act_dtype"), ("m", 0, "m, n and k"), ("k", 1 << 21, "m, n and k"),
                                ("x_eps", math.nan, "x_eps"), ("x_eps", -1.0, "x_eps"), ("w", 40, "16-byte"), ("x", None, "non-NULL"),
                                ("x_row_stride", 39, "row strides"), ("out_row_stride", 7, "row strides"),
                                ("act_dtype", 0, "workspace too small")):
        bad = N.Linear4Args.from_buffer_copy(a)
        setattr(bad, field, value)
        refused_c(lib.uttt_linear4, bad, match)
    a = N.Readout4Args(batch=1, tokens=1, d_model=64, d_ff=64, act_dtype=0, eps=1e-5, x=16, w_up=16, w_gate=16, w_down=16,
                       ln_weight=16, ln_bias=16, out=16, workspace=16, workspace_bytes=lib.uttt_readout4_workspace(1, 1, 64, 64))
    for field, value, match in (("d_model", 4160, "multiples of 64"), ("d_ff", 100, "multiples of 64"), ("batch", 0, "batch"),
                                ("eps", 0.0, "eps"), ("workspace_bytes", 8, "workspace too small"), ("workspace", None, "workspace"),
                                ("x_stride_b", 3, "16-byte"), ("w_up_stride", 8, "16-byte"), ("ln_bias", None, "non-NULL")):
        bad = N.Readout4Args.from_buffer_copy(a)
        setattr(bad, field, value)
        refused_c(lib.uttt_readout4, bad, match)
    a = N.SwaTree4Args(n_req=1, n_heads=4, n_kv_heads=2, nodes=1, head_dim=64, window=4096, sinks=0, act_dtype=1, scale=0.1,
                       positions=16, q=16, k_new=16, v_new=16, cache=16, out=16)
    for field, value, match in (("head_dim", 96, "head_dim"), ("nodes", 65, "nodes"), ("n_kv_heads", 3, "head counts"), ("window", 0, "window"),
                                ("scale", 0.0, "scale"), ("k_nodes", 16, "pairs"), ("sin_table", 16, "both"), ("cache", 24, "16-byte"),
                                ("q_stride_t", 4, "16-byte"), ("positions", None, "non-NULL"), ("scale", 0.2, "workspace too small")):
        bad = N.SwaTree4Args.from_buffer_copy(a)
        setattr(bad, field, value)
        refused_c(lib.uttt_swa_tree4, bad, match)
    a = N.KvCommit4Args(layers=2, n_req=2, n_kv_heads=1, n_nodes=3, path=3, head_dim=64, window=32, sinks=0, act_dtype=1, k_nodes=16,
                        v_nodes=16, cache=16, cache_stride_l=4608, cache_stride_n=2304, positions=16)
    for field, value, match in (("layers", 0, "out of range"), ("n_req", 70000, "out of range"), ("head_dim", 32, "head_dim"),
                                ("window", 0, "window"), ("cache", 8, "16-byte"), ("cache_stride_n", 0, "overlap"),
                                ("cache_stride_l", 2304, "overlap"), ("path", 4, "path"), ("k_nodes", None, "non-NULL"),
                                ("nodes_stride_h", 4, "16-byte"), ("act_dtype", 7, "act_dtype")):
        bad = N.KvCommit4Args.from_buffer_copy(a)
        setattr(bad, field, value)
        refused_c(lib.uttt_kv_commit4, bad, match)
    a = N.KvFork4Args(layers=1, n_req=129, n_kv_heads=1, head_dim=64, window=32, sinks=0, sources=16, cache=16, cache_stride_n=2304)
    refused_c(lib.uttt_kv_fork4, a, "at most 128")
    a = N.KvValues4Args(layers=1, n_req=1, n_kv_heads=1, head_dim=64, window=32, sinks=0, act_dtype=1, cache=16, k=16)
    refused_c(lib.uttt_kv_values4, a, "non-NULL")
    a = N.BeamSelectArgs(rows=4, vocab=100, beams=2, dtype=1, logits=16, row_stride=100, scores=16, tokens=16, sources=16, out_scores=16,
                         workspace=16, workspace_bytes=lib.uttt_beam_select_workspace(4, 100, 2))
    for field, value, match in (("beams", 3, "multiple of beams"), ("beams", 33, "beams must be"), ("vocab", 0, "vocab"), ("pad", 100, "pad"),
                                ("n_banned", 9, "at most 8"), ("row_stride", 99, "row stride"), ("workspace_bytes", 10, "workspace"),
                                ("scores", None, "non-NULL"), ("dtype", 5, "bad dtype")):
        bad = N.BeamSelectArgs.from_buffer_copy(a)
        setattr(bad, field, value)
        refused_c(lib.uttt_beam_select, bad, match)
    for size in (lib.uttt_readout4_workspace(0, 1, 64, 64), lib.uttt_swa_tree4_workspace(0, 1, 1, 1, 64, 1, 0),
                 lib.uttt_beam_select_workspace(1, 0, 1)):
        assert size == 0
