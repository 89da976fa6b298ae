"""Host side of the serving operators (no GPU needed: every case is rejected before any device call): the C
header's declarations and layouts, refusals of the wrappers (ValueError) and of the C ABI (a status with a message)."""
import ctypes as C
import hashlib
import os
import re
import subprocess

import pytest
import torch

from utttcompanion_amd import _native as N
from utttcompanion_amd import build
from utttcompanion_amd import kernels as K

STRUCTS = {"uttt_sample_args": N.SampleArgs, "uttt_swa_tree_args": N.SwaTreeArgs, "uttt_kv_commit_args": N.KvCommitArgs,
           "uttt_kv_fork_args": N.KvForkArgs}


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(build.LIB_PATH):
        build.build()
    return N.load_library()


def test_every_declared_symbol_is_exported_and_typed(lib):
    text = re.sub(r"/\*.*?\*/", "", open(N.SERVE_HEADER_PATH).read(), flags=re.S)
    names = set(re.findall(r"\b(uttt_[a-z0-9_]+)\s*\(", text))
    assert names == set(N.SERVE_SIGNATURES)
    assert all(hasattr(lib, name) for name in names)
    assert lib.uttt_serve_abi_version() == N.SERVE_ABI_VERSION


def test_declarations_belong_to_the_abi_version():
    """Other declarations take another UTTT_SERVE_ABI_VERSION: the digest changes together with it."""
    text = re.sub(r"/\*.*?\*/", " ", open(N.SERVE_HEADER_PATH).read(), flags=re.S)
    text = " ".join(re.sub(r"#define UTTT_SERVE_ABI_VERSION \d+", "", text).split())
    assert (N.SERVE_ABI_VERSION, hashlib.sha256(text.encode()).hexdigest()[:16]) == (1, "0570f8f0508d4549")


@pytest.mark.parametrize("serve", ["", "int uttt_serve_abi_version(void) { return 0; }"])
def test_library_without_these_entry_points_is_refused(tmp_path, monkeypatch, serve):
    (tmp_path / "old.c").write_text(f"int uttt_abi_version(void) {{ return {N.ABI_VERSION}; }}\n{serve}\n")
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(tmp_path / "old.so"), str(tmp_path / "old.c")], check=True)
    monkeypatch.setattr(N, "_lib", None)
    with pytest.raises(RuntimeError, match="serving ABI version 0, expected"):
        N.load_library(str(tmp_path / "old.so"))


def test_struct_layouts_match_the_c_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{N.SERVE_HEADER_PATH}"', 'int main(void) {']
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


def test_packed_arguments_are_the_structure():
    """The wrappers pack the blocks by ``struct``: the same bytes as the ctypes structure's."""
    a = N.KvForkArgs(2, 3, 4, 5, 64, 1, 0x1000, 0x2000, 0x3000, 7, 8, 0x4000)
    assert N.pack_kv_fork(2, 3, 4, 5, 64, 1, 0x1000, 0x2000, 0x3000, 7, 8, 0x4000) == bytes(a)
    s = N.SampleArgs(rows=2, vocab=10, dtype=1, n_banned=1, banned=(C.c_int32 * 8)(3), active_limit=-1, logits=16,
                     row_stride=10, uniforms=32, temperature=48, top_k=0, top_p=64, min_p=0, out=80, logprob=96, advance=0)
    assert N.pack_sample(2, 10, 1, 1, 3, 0, 0, 0, 0, 0, 0, 0, -1, 16, 10, 32, 48, 0, 64, 0, 80, 96, 0) == bytes(s)


# ---------------------------------------------------------------------------- the wrappers
def refused(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def test_sample_select_refusals():
    x, u = torch.zeros(2, 100), torch.zeros(2)
    refused("rows, vocab", K.sample_select, torch.zeros(100), u, u)
    refused("unit column stride", K.sample_select, torch.zeros(100, 2).t(), u, u)
    refused("at most 8", K.sample_select, x, u, u, banned=range(9))
    refused("2\\^20", K.sample_select, torch.zeros(2, 0), u, u)
    refused("2\\^20", K.sample_select, torch.zeros(1, (1 << 20) + 1), u[:1], u[:1])
    refused("", K.sample_select, x.half(), u, u)
    refused("uniforms", K.sample_select, x, torch.zeros(3), u)
    refused("uniforms", K.sample_select, x, u.double(), u)
    refused("temperature", K.sample_select, x, u, torch.zeros(1).expand(2))
    refused("top_k", K.sample_select, x, u, u, top_k=torch.zeros(2, dtype=torch.int64))
    refused("top_p", K.sample_select, x, u, u, top_p=torch.zeros(2, 1))
    refused("min_p", K.sample_select, x, u, u, min_p=torch.zeros(2, dtype=torch.bfloat16))
    refused("advance", K.sample_select, x, u, u, advance=torch.zeros(2, dtype=torch.int32))
    refused("no CPU path", K.sample_select, x, u, u)


def tree(n=2, t=3, heads=4, hkv=2, hd=64, slots=20, dtype=torch.bfloat16):
    z = lambda *shape: torch.zeros(shape, dtype=dtype)
    return [z(n, t, heads, hd), z(n, t, hkv, hd), z(n, t, hkv, hd), z(n, hkv, slots, hd), z(n, hkv, slots, hd),
            torch.zeros(n, dtype=torch.int64)]


def test_swa_tree_refusals():
    good = tree()
    with_ = lambda **at: [at.get(f"a{i}", a) for i, a in enumerate(good)]
    refused("must be \\(N, T, H, hd\\)", K.swa_tree, *with_(a0=good[0][:, 0]))
    refused("1 to 64 nodes", K.swa_tree, *tree(t=65))
    refused("1 to 64 nodes", K.swa_tree, *tree(t=0))
    refused("head_dim", K.swa_tree, *tree(hd=96))
    refused("multiple", K.swa_tree, *tree(heads=5))
    refused("sinks", K.swa_tree, *good, sinks=20)
    refused("sinks", K.swa_tree, *good, sinks=-1)
    refused("new keys", K.swa_tree, *with_(a1=good[1][:, :2]))
    refused("new keys", K.swa_tree, *with_(a3=good[3][:1], a4=good[4][:1]))
    refused("share one dtype", K.swa_tree, *with_(a1=good[1].float()))
    refused("rings must be two", K.swa_tree, *with_(a4=good[4][:, :, :19]))
    refused("rings must be contiguous|contiguous and 16-byte", K.swa_tree,
            *with_(a3=torch.zeros(2, 2, 20, 128, dtype=torch.bfloat16)[..., :64], a4=torch.zeros(2, 2, 20, 128, dtype=torch.bfloat16)[..., :64]))
    refused("positions", K.swa_tree, *with_(a5=good[5].int()))
    refused("parents", K.swa_tree, *good, parents=torch.zeros(2, 3, dtype=torch.int64))
    refused("parents", K.swa_tree, *good, parents=torch.zeros(2, 2, dtype=torch.int32))
    refused("counts", K.swa_tree, *good, counts=torch.zeros(2, dtype=torch.int64))
    refused("both be given", K.swa_tree, *good, cos=torch.zeros(9, 64))
    refused("tables", K.swa_tree, *good, cos=torch.zeros(9, 64), sin=torch.zeros(8, 64))
    refused("tables", K.swa_tree, *good, cos=torch.zeros(9, 64).half(), sin=torch.zeros(9, 64).half())
    refused("no CPU path", K.swa_tree, *good)
    q, k, v = (a[:, 0] for a in good[:3])
    refused("sinks", K.swa_decode, q, k, v, *good[3:], sinks=-1)
    refused("new keys", K.swa_decode, q, k[:1], v, *good[3:], sinks=2)
    refused("sinks", K.swa_prefill, *(a.transpose(1, 2) for a in good[:3]), 5, 0, sinks=-1)
    refused("sinks", K.swa_prefill, *(a.transpose(1, 2) for a in good[:3]), 5, 0, sinks=2, build_only=True)


def test_kv_copy_refusals():
    _, kn, vn, kr, vr, pos = tree()
    ids, counts = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    refused("rings must be two", K.kv_commit, kn, vn, ids, counts, kr, vr[:, :1], pos)
    refused("one row per ring", K.kv_commit, kn[:, :, :1], vn, ids, counts, kr, vr, pos)
    refused("one dtype", K.kv_commit, kn.float(), vn, ids, counts, kr, vr, pos)
    refused("sinks", K.kv_commit, kn, vn, ids, counts, kr, vr, pos, sinks=20)
    refused("nodes must be int32", K.kv_commit, kn, vn, ids.long(), counts, kr, vr, pos)
    refused("nodes must be int32", K.kv_commit, kn, vn, ids.t().contiguous().t(), counts, kr, vr, pos)
    refused("counts", K.kv_commit, kn, vn, ids, counts[:1], kr, vr, pos)
    refused("positions", K.kv_commit, kn, vn, ids, counts, kr, vr, pos.int())
    refused("no CPU path", K.kv_commit, kn, vn, ids, counts, kr, vr, pos)
    refused("whole 16-byte pieces", K.kv_fork, kr[..., :4].contiguous(), vr[..., :4].contiguous(), counts, pos)
    refused("at most 128", K.kv_fork, *(torch.zeros(129, 1, 1, 64) for _ in range(2)), counts, pos)
    refused("sources", K.kv_fork, kr, vr, counts.long(), pos)
    refused("no CPU path", K.kv_fork, kr, vr, counts, pos)


# ---------------------------------------------------------------------------- the C ABI
def _fake(n):  # aligned, never dereferenced: every call below fails its checks first
    return 0x100000 + 0x1000 * n


def fails(lib, fn, args, message, **changes):
    for name, value in changes.items():
        setattr(args, name, value)
    assert getattr(lib, fn)(bytes(args), None) == 1
    assert message in lib.uttt_last_error(), lib.uttt_last_error()


def test_c_abi_refuses_bad_samples(lib):
    def args():
        return N.SampleArgs(rows=2, vocab=100, dtype=N.DTYPE_F32, active_limit=-1, logits=_fake(1), row_stride=100,
                            uniforms=_fake(2), temperature=_fake(3), out=_fake(4))
    for changes, message in ((dict(rows=0), b"rows"), (dict(rows=65536), b"rows"), (dict(vocab=0), b"vocab"),
                             (dict(vocab=(1 << 20) + 1), b"vocab"), (dict(dtype=7), b"bf16 or fp32"),
                             (dict(n_banned=9), b"at most 8"), (dict(n_banned=-1), b"at most 8"),
                             (dict(n_banned=1, banned=(C.c_int32 * 8)(-1)), b">= 0"), (dict(logits=0), b"non-NULL"),
                             (dict(out=0), b"non-NULL"), (dict(row_stride=99), b"row stride")):
        fails(lib, "uttt_sample_select", args(), message, **changes)
    assert lib.uttt_sample_select(None, None) == 1


def test_c_abi_refuses_bad_trees(lib):
    def args():
        return N.SwaTreeArgs(n_req=2, n_heads=4, n_kv_heads=2, nodes=3, head_dim=64, window=18, sinks=2, act_dtype=N.DTYPE_BF16,
                             scale=0.125, positions=_fake(1), q=_fake(2), q_stride_n=768, q_stride_t=256, q_stride_h=64,
                             k_new=_fake(3), k_stride_n=384, k_stride_t=128, k_stride_h=64, v_new=_fake(4), v_stride_n=384,
                             v_stride_t=128, v_stride_h=64, k_ring=_fake(5), v_ring=_fake(6), ring_stride_n=2560, out=_fake(7),
                             o_stride_n=768, o_stride_t=256, o_stride_h=64, k_nodes=_fake(8), v_nodes=_fake(9))
    for changes, message in ((dict(head_dim=80), b"head_dim"), (dict(n_req=0), b"request / head"), (dict(n_heads=5), b"head counts"),
                             (dict(nodes=0), b"nodes"), (dict(nodes=65), b"nodes"), (dict(window=0), b"window"),
                             (dict(sinks=-1), b"window or sinks"), (dict(window=1 << 23), b"2 GB"), (dict(act_dtype=9), b"act_dtype"),
                             (dict(scale=0.0), b"scale"), (dict(positions=0), b"non-NULL"), (dict(v_nodes=0), b"pairs"),
                             (dict(write_ring=1), b"write_ring"), (dict(cos_table=_fake(10)), b"both"), (dict(q=_fake(2) + 8), b"16-byte"),
                             (dict(k_stride_t=130), b"16-byte"),
                             (dict(write_ring=1, nodes=1, k_nodes=0, v_nodes=0, ring_stride_n=0), b"overlap"),
                             (dict(window=1 << 16), b"workspace")):
        fails(lib, "uttt_swa_tree", args(), message, **changes)
    assert lib.uttt_swa_tree(None, None) == 1
    assert lib.uttt_swa_tree_workspace(0, 4, 2, 3, 64, 20, N.DTYPE_BF16) <= 16
    p = N.SwaPrefillArgs()
    assert lib.uttt_swa_prefill_sinks(C.byref(p), -1, None) == 1 and b"sinks" in lib.uttt_last_error()


def test_c_abi_refuses_bad_copies(lib):
    def commit():
        return N.KvCommitArgs(layers=2, n_req=2, n_kv_heads=2, n_nodes=3, path=3, head_dim=64, window=18, sinks=2,
                              act_dtype=N.DTYPE_BF16, k_nodes=_fake(1), v_nodes=_fake(2), nodes_stride_l=768, nodes_stride_n=384,
                              nodes=_fake(3), path_stride=3, counts=_fake(4), k_ring=_fake(5), v_ring=_fake(6),
                              ring_stride_l=5120, ring_stride_n=2560, positions=_fake(7))
    for changes, message in ((dict(layers=0), b"layers"), (dict(n_req=0), b"requests"), (dict(n_nodes=0), b"node"),
                             (dict(path=0), b"path"), (dict(window=0), b"window"), (dict(act_dtype=5), b"act_dtype"),
                             (dict(head_dim=4), b"pieces"), (dict(counts=0), b"non-NULL"), (dict(k_ring=_fake(5) + 4), b"16-byte"),
                             (dict(ring_stride_n=2564), b"pieces"), (dict(ring_stride_n=0), b"overlap"),
                             (dict(ring_stride_l=2560), b"overlap"), (dict(ring_stride_l=0), b"overlap")):
        fails(lib, "uttt_kv_commit", commit(), message, **changes)

    def fork():
        return N.KvForkArgs(layers=2, n_req=2, n_kv_heads=2, slots=20, head_dim=64, act_dtype=N.DTYPE_BF16, sources=_fake(1),
                            k_ring=_fake(2), v_ring=_fake(3), ring_stride_l=5120, ring_stride_n=2560, positions=_fake(4))
    for changes, message in ((dict(layers=0), b"layers"), (dict(n_req=129), b"at most 128"), (dict(slots=0), b"slot"),
                             (dict(act_dtype=5), b"act_dtype"), (dict(head_dim=12), b"pieces"), (dict(sources=0), b"non-NULL"),
                             (dict(ring_stride_l=5124), b"pieces"), (dict(ring_stride_n=1280), b"overlap"),
                             (dict(ring_stride_l=2560, ring_stride_n=2560), b"overlap")):
        fails(lib, "uttt_kv_fork", fork(), message, **changes)


def test_configuration_and_layer_take_sinks():
    from utttcompanion_amd import uTTTConfig
    from utttcompanion_amd.layer import SlidingWindowAttention, history_rows, kept_rows
    assert uTTTConfig().attention_sinks == 0
    assert uTTTConfig.from_dict({"model": {"attention_sinks": 4}}).attention_sinks == 4
    with pytest.raises(ValueError, match="sinks"):
        SlidingWindowAttention(64, 4, 2, sinks=-1)
    rows = torch.arange(12.0).view(1, 1, 12, 1)
    assert kept_rows(rows, 4, 3).flatten().tolist() == [0, 1, 2, 8, 9, 10, 11]
    assert kept_rows(rows, 4, 0).flatten().tolist() == [8, 9, 10, 11]
    assert kept_rows(rows, 9, 3) is rows
    assert [history_rows(c, 4, 3) for c in (0, 2, 3, 5, 6, 7)] == [(0, 0), (2, 0), (3, 0), (3, 2), (3, 3), (3, 3)]
    assert [history_rows(c, 4, 0) for c in (0, 3, 4)] == [(0, 0), (0, 3), (0, 3)]
    assert history_rows(5, 1, 2) == (2, 0)
