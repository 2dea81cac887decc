"""CPU checks of the low-bit decode step's boundary: struct layouts, refusals before any launch, the 4-bit layout, the decoder's choices."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest
import torch

from physicedit_amd import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF = torch.bfloat16
STRUCTS = {"pe_w4_weight": L.W4Weight, "pe_kv_cache": L.KvCache, "pe_kv_append_args": L.KvAppendArgs, "pe_logits_args": L.LogitsArgs}


@pytest.fixture(scope="module")
def lib():
    from physicedit_amd import build
    if not os.path.exists(L.LIB_PATH):
        build.build(verbose=False)
    return L.lib()


def refused(lib, rc, text):
    assert rc == -1 and re.search(text, lib.pe_last_error().decode()), (rc, lib.pe_last_error())


def test_struct_layouts(tmp_path):
    """every field of the new structs at the C compiler's offset"""
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "physicedit_amd.h"', "int main(void) {"]
    for name, cls in STRUCTS.items():
        lines.append(f'  printf("{name} %zu", sizeof({name}));')
        lines += [f'  printf(" %zu", offsetof({name}, {f[0]}));' for f in cls._fields_] + ['  printf("\\n");']
    (tmp_path / "a.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "a.c"), "-o", str(tmp_path / "a")], check=True)
    for line in subprocess.run([str(tmp_path / "a")], check=True, capture_output=True, text=True).stdout.splitlines():
        name, size, *offsets = line.split()
        assert C.sizeof(STRUCTS[name]) == int(size) and [getattr(STRUCTS[name], f[0]).offset for f in STRUCTS[name]._fields_] == [int(o) for o in offsets], name


P = 1 << 20          # an address that is never read: every call below is refused on the host


def w4(N=32, K=256, group=128, codes=P, scale=P):
    return L.W4Weight(codes, scale, N, K, group)


@pytest.mark.parametrize("kw,args,text", [
    (dict(codes=None), {}, "null"), (dict(scale=None), {}, "null"), (dict(group=96), {}, "group of 96"), (dict(K=200), {}, "multiple of the group"),
    (dict(N=0), {}, "N=0"), ({}, dict(M=0), "M=0"), ({}, dict(M=65), "M=65"), ({}, dict(x=None), "null"), ({}, dict(out=None), "null"),
    ({}, dict(ldx=248), "aligned"), ({}, dict(ldx=260), "aligned"), ({}, dict(x=P + 8), "aligned"), (dict(codes=P + 4), {}, "unaligned"),
    ({}, dict(ldo=31), "row stride"), ({}, dict(res=P, ldr=31), "row stride"), (dict(N=48), dict(swiglu=1), "gated"), ({}, dict(swiglu=1, res=P), "residual"),
    (dict(N=1 << 27), dict(ldo=1 << 28), "out of range"), ({}, dict(out=P), "not x")])
def test_gemv_w4_refusals(lib, kw, args, text):
    a = dict(x=P, ldx=256, M=1, bias=None, res=None, ldr=32, out=2 * P, ldo=32, swiglu=0, eps=-1.0) | args
    refused(lib, lib.pe_gemv_w4(a["x"], a["ldx"], a["M"], C.byref(w4(**kw)), a["bias"], a["res"], a["ldr"], a["out"], a["ldo"], a["swiglu"], a["eps"], None), text)


def test_gemv_w4_null_weight(lib):
    refused(lib, lib.pe_gemv_w4(P, 256, 1, None, None, None, 0, 2 * P, 32, 0, -1.0, None), "null weight")


def cache(k=P, v=P, ks=P, vs=P, batch=2, n_kv=2, capacity=128, head_dim=128):
    return L.KvCache(k, v, ks, vs, batch, n_kv, capacity, head_dim)


@pytest.mark.parametrize("kw,args,text", [
    (dict(k=None), {}, "null"), (dict(vs=None), {}, "null"), ({}, dict(k=None), "null"), ({}, dict(start=None), "null"), (dict(head_dim=96), {}, "heads of 96"),
    (dict(capacity=100), {}, "bad shape"), (dict(capacity=0), {}, "bad shape"), (dict(batch=0), {}, "bad shape"), ({}, dict(T=0), "bad shape"),
    ({}, dict(cos=P), "come together"), ({}, dict(cos=P, sin=P, table_rows=0), "come together"), ({}, dict(n_q=4, q=P, q_out=P), "queries are rotated"),
    ({}, dict(positions=P), "positions"), ({}, dict(k=P + 2), "aligned"), ({}, dict(v_strides=(4, 8, 8)), "strides"),
    (dict(batch=70000), {}, "too many")])
def test_kv_append_refusals(lib, kw, args, text):
    a = dict(q=None, k=P, v=P, q_strides=(0, 0, 0), k_strides=(512, 256, 128), v_strides=(512, 256, 128), q_out=None, cos=None, sin=None, table_rows=8,
             table_f32=0, positions=None, start=P, T=2, n_q=0) | args
    refused(lib, lib.pe_kv_append_e4m3(C.byref(cache(**kw)), C.byref(L.KvAppendArgs(*(a[f[0]] for f in L.KvAppendArgs._fields_))), None), text)


@pytest.mark.parametrize("kw,args,text", [
    (dict(k=None), {}, "null"), ({}, dict(q=None), "null"), ({}, dict(out=None), "null"), ({}, dict(start=None), "null"), (dict(head_dim=80), {}, "heads of 80"),
    (dict(capacity=96), {}, "bad shape"), ({}, dict(n_q=3), "bad shape"), ({}, dict(n_q=0), "bad shape"), ({}, dict(T=0), "T=0"), ({}, dict(T=65), "T=65"),
    ({}, dict(q=P + 8), "aligned"), ({}, dict(tree=P + 4), "aligned"), ({}, dict(strides=(8, 8, 12)), "strides"), (dict(capacity=1024), dict(ws=None), "workspace"),
    (dict(capacity=1024), dict(nbytes=100), "workspace"), (dict(n_kv=70000), dict(n_q=70000), "too many")])
def test_kv_attention_refusals(lib, kw, args, text):
    a = dict(q=P, strides=(1024, 512, 128), start=P, tree=None, T=2, n_q=4, out=P, ws=P, nbytes=1 << 40) | args
    refused(lib, lib.pe_kv_attention_e4m3(C.byref(cache(**kw)), a["q"], (C.c_longlong * 3)(*a["strides"]), a["start"], a["tree"], a["T"], a["n_q"], 0.1, a["out"],
                                          a["ws"], a["nbytes"], None), text)


def test_null_arguments(lib):
    refused(lib, lib.pe_kv_append_e4m3(None, None, None), "null argument")
    refused(lib, lib.pe_kv_attention_e4m3(None, P, None, P, None, 1, 1, 0.1, P, P, 1, None), "null argument")
    refused(lib, lib.pe_process_logits(None, P, None), "null argument")
    refused(lib, lib.pe_select_token(None, P, 0, None, None, 0, P, 1, None), "null argument")


def test_workspace_sizes(lib):
    """a long cache is split, a short one is not; shapes that no call takes need nothing"""
    assert lib.pe_kv_attention_workspace_bytes(1, 4, 1, 28, 128, 64) == 0
    assert lib.pe_kv_attention_workspace_bytes(1, 4, 1, 28, 128, 15360) >= 2 * 28 * 130 * 4
    assert lib.pe_kv_attention_workspace_bytes(0, 4, 1, 28, 128, 15360) == 0
    assert lib.pe_select_token_workspace_bytes(3, 152064) == 3 * 75 * 8 and lib.pe_select_token_workspace_bytes(0, 5) == 0
    assert lib.pe_select_token_workspace_bytes(3, 8192) == 0 and lib.pe_select_token_workspace_bytes(1, 8193) == 5 * 8


@pytest.mark.parametrize("args,text", [
    (dict(logits=None), "null"), (dict(rows=0), "bad shape"), (dict(vocab=0), "bad shape"), (dict(rows=70000), "bad shape"), (dict(ld=99), "row stride"),
    (dict(logits=P + 1), "unaligned"), (dict(logits=P + 2, f32=1), "unaligned"), (dict(penalties=P), "need the counts"),
    (dict(counts=P, ld_counts=99), "counts"), (dict(bias=P, ld_bias=99), "bias"), (dict(allowed=P, ld_allowed=3), "mask")])
def test_logits_refusals(lib, args, text):
    a = dict(logits=P, ld=100, f32=0, rows=2, vocab=100, counts=None, ld_counts=0, penalties=None, ld_penalties=0, bias=None, ld_bias=0, allowed=None,
             ld_allowed=0) | args
    s = L.LogitsArgs(*(a[f[0]] for f in L.LogitsArgs._fields_))
    refused(lib, lib.pe_process_logits(C.byref(s), P, None), text)
    refused(lib, lib.pe_select_token(C.byref(s), P, 0, None, None, 0, P, 1 << 20, None), text)


def test_select_and_counts_refusals(lib):
    s = L.LogitsArgs(logits=P, ld=100, rows=2, vocab=100)
    refused(lib, lib.pe_process_logits(C.byref(s), None, None), "null")
    refused(lib, lib.pe_select_token(C.byref(s), None, 0, None, None, 0, P, 1 << 20, None), "null token")
    refused(lib, lib.pe_select_token(C.byref(s), P, 1, None, None, 0, P, 1 << 20, None), "no counts")
    refused(lib, lib.pe_select_token(C.byref(s), P, 0, P, P, 8, P, 1 << 20, None), "one row")
    big = L.LogitsArgs(logits=P, ld=100000, rows=2, vocab=100000)
    refused(lib, lib.pe_select_token(C.byref(big), P, 0, None, None, 0, P, 8, None), "workspace of 784")
    refused(lib, lib.pe_token_counts_add(None, 100, 2, 100, P, 3, 0, None), "null")
    refused(lib, lib.pe_token_counts_add(P, 99, 2, 100, P, 3, 0, None), "bad shape")
    refused(lib, lib.pe_token_counts_add(P, 100, 2, 100, P, 0, 0, None), "bad shape")


def test_operators_have_no_cpu_path():
    from physicedit_amd import ops
    x = torch.zeros((2, 128), dtype=BF)
    for call in (lambda: ops.pack_w4(torch.zeros((16, 64), dtype=torch.uint8), torch.zeros((16, 1), dtype=BF)), lambda: ops.quantize_w4(x),
                 lambda: ops.process_logits(x), lambda: ops.select_token(x), lambda: ops.token_counts_add(torch.zeros((1, 8), dtype=torch.int16), torch.zeros((1, 1), dtype=torch.int32)),
                 lambda: ops.kv_append_e4m3(ops.KVCacheE4M3(1, 1, 64, 64, device="cpu"), x, x, x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("N,K,group", [(37, 416, 32), (16, 128, 128), (1, 64, 64), (50, 640, 128)])
def test_pack_w4_layout(monkeypatch, N, K, group):
    """the tiles as include/physicedit_amd.h lays them down, word by word"""
    from physicedit_amd import ops
    monkeypatch.setattr(ops, "_stream_of", lambda dev, name: 0)
    monkeypatch.setattr(ops, "_at", lambda t, *a: None)
    g = torch.Generator().manual_seed(N)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scale, zero = torch.rand((N, K // group), generator=g).to(BF), torch.randint(0, 16, (N, K // group), generator=g, dtype=torch.uint8)
    for z in (zero, None):
        w = ops.pack_w4(codes, scale, z, group)
        words = w.codes.contiguous().view(torch.int32)                       # [tiles, chunks, 64, 4]
        tiles, chunks = (N + 15) // 16, (K + 127) // 128
        assert words.shape == (tiles, chunks, 64, 4)
        plain = torch.zeros((tiles * 16, chunks * 128), dtype=torch.int32)
        plain[:N, 0:K:2], plain[:N, 1:K:2] = (codes & 15).int(), (codes >> 4).int()
        for lane in range(64):
            for s in range(4):
                for e in range(8):
                    got = (words[:, :, lane, s] >> (4 * (e // 2 + 4 * (e % 2)))) & 15
                    k = 32 * s + 8 * (lane // 16) + e
                    assert torch.equal(got, plain.view(tiles, 16, chunks, 128)[:, lane % 16, :, k])
        pair = w.scale.view(tiles, -1, 16, 2).transpose(1, 2).reshape(tiles * 16, -1, 2)
        assert torch.equal(pair[:N, :K // group, 0], scale)
        assert torch.equal(pair[:N, :K // group, 1].float(), -128.0 - (zero.float() if z is not None else torch.full((N, K // group), 8.0)))
        assert not pair[N:].any() and not pair[:, K // group:].any()
        assert w.nbytes == tiles * chunks * 1024 + pair.numel() * 2


def test_weights_and_caches_hold_their_buffers():
    """the structs passed to the kernels hold addresses: parts of another shape are refused, and the buffers behind the addresses cannot be exchanged"""
    from physicedit_amd import ops
    codes, scale = torch.zeros((3, 2, 64, 16), dtype=torch.uint8), torch.zeros((3, 8, 16, 2), dtype=BF)
    w = ops.W4Weight(codes, scale, 33, 256, 32)
    assert w.codes is codes and w.scale is scale
    for args in ((codes[:2], scale, 33, 256, 32), (codes, scale[:2], 33, 256, 32), (codes, scale, 49, 256, 32), (codes, scale, 33, 260, 32), (codes, scale, 33, 288, 32),
                 (codes, scale, 33, 256, 64), (codes, scale, 33, 256, 16), (codes.char(), scale, 33, 256, 32), (codes, scale.half(), 33, 256, 32),
                 (codes.transpose(0, 1).contiguous().transpose(0, 1), scale, 33, 256, 32), (codes, scale.to("meta"), 33, 256, 32), (codes, scale, 0, 256, 32)):
        with pytest.raises(ValueError, match="W4Weight"):
            ops.W4Weight(*args)
    cache = ops.KVCacheE4M3(1, 2, 64, 64, device="cpu")
    for obj, names in ((w, ("codes", "scale", "N", "K", "group")), (cache, ("k", "v", "k_scale", "v_scale", "batch", "n_kv", "capacity", "head_dim"))):
        for name in names:
            with pytest.raises(AttributeError):
                setattr(obj, name, getattr(obj, name))


def test_gemv_w4_eps_is_a_number(lib):
    """a NaN is not "no norm" """
    refused(lib, lib.pe_gemv_w4(P, 256, 1, C.byref(w4()), None, None, 32, 2 * P, 32, 0, float("nan"), None), "norm_eps")


def test_pack_w4_zero_points_are_codes(monkeypatch):
    """a zero point above 15 is refused, not cut to four bits"""
    from physicedit_amd import ops
    monkeypatch.setattr(ops, "_stream_of", lambda dev, name: 0)
    monkeypatch.setattr(ops, "_at", lambda t, *a: None)
    codes, scale = torch.zeros((16, 64), dtype=torch.uint8), torch.ones((16, 1), dtype=BF)
    zero = torch.full((16, 1), 15, dtype=torch.uint8)
    assert float(ops.pack_w4(codes, scale, zero).scale[0, 0, 3, 1]) == -143
    zero[7] = 16
    with pytest.raises(ValueError, match="above 15"):
        ops.pack_w4(codes, scale, zero)
