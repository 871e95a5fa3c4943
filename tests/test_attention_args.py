"""What the paged-cache and prompt attention entries refuse, before anything is launched: no GPU needed."""
import pytest
import torch

from fuel_b200 import _lib as L, ops

F32, F16, BF16, Q4K = 0, 1, 30, 12
A = 4096   # an aligned address that nothing is read from: every call below is refused first


def append(act=F32, cache=F32, k=A, ks=1024, v=A, vs=1024, q=A, qs=4096, q_out=2 * A, k_out=None, kc=A, vc=A, table=A, seq=A, pos=A,
           cos=A, sin=A, rows=4, seqs=4, heads=32, kv=8, hd=128, page=16, pages=8, width=2, max_pos=64):
    return L.lib.fuelq_paged_append(act, cache, k, ks, v, vs, q, qs, q_out, k_out, kc, vc, table, seq, pos, cos, sin, rows, seqs, heads,
                                    kv, hd, page, pages, width, max_pos, None)


def decode(scale=0.1, act=F32, cache=F32, q=A, qs=4096, kc=A, vc=A, out=A, table=A, lens=A, seqs=4, heads=32, kv=8, hd=128, page=16, pages=8,
           width=2, ws=A, ws_bytes=1 << 40):
    return L.lib.fuelq_paged_attn_decode(act, cache, q, qs, kc, vc, out, table, lens, seqs, heads, kv, hd, page, pages, width, scale, ws,
                                         ws_bytes, None)


def prompt(scale=0.1, act=F32, q=A, qs=4096, k=A, ks=1024, v=A, vs=1024, out=A, cu=A, seqs=4, rows=64, heads=32, kv=8, hd=128, ws=A,
           ws_bytes=1 << 40):
    return L.lib.fuelq_prompt_attn(act, q, qs, k, ks, v, vs, out, cu, seqs, rows, heads, kv, hd, scale, ws, ws_bytes, None)


@pytest.mark.parametrize("call", [append, decode])
def test_types_and_sizes_of_the_cache(call):
    for pair in ((Q4K, F32), (F32, Q4K), (F16, BF16), (BF16, F16), (F16, F32), (BF16, F32)):
        assert call(act=pair[0], cache=pair[1]) == L.NOT_SUPPORTED, pair
    for hd in (0, 32, 80, 96, 256):
        assert call(hd=hd) == L.NOT_SUPPORTED
    for page in (0, -16, 3, 24, 2048):
        assert call(page=page) == L.NOT_SUPPORTED
    assert call(heads=30) == L.INVALID_PROBLEM      # 8 kv heads
    assert call(kv=0) == L.INVALID_PROBLEM
    assert call(heads=0) == L.INVALID_PROBLEM
    assert call(pages=-1) == L.INVALID_PROBLEM
    assert call(width=-1) == L.INVALID_PROBLEM
    assert call(seqs=-1) == L.INVALID_PROBLEM


def test_append_refusals():
    assert append(rows=0) == L.OK and append(rows=0, k=None, kc=None) == L.OK
    assert append(rows=-1) == L.INVALID_PROBLEM and append(rows=1 << 31) == L.INVALID_PROBLEM
    for name in ("k", "v", "kc", "vc", "table", "pos", "cos", "sin", "q_out"):
        assert append(**{name: None}) == L.INVALID_PROBLEM, name
    assert append(seq=None, rows=5) == L.INVALID_PROBLEM          # row t is sequence t: more rows than sequences
    for name in ("k", "v", "q", "q_out", "k_out", "kc", "vc", "cos", "sin"):
        assert append(**{name: A + 8}) == L.MISALIGNED, name
    assert append(ks=1023) == L.INVALID_PROBLEM and append(ks=1026) == L.INVALID_PROBLEM   # overlapping rows; not 16 bytes
    assert append(vs=1000) == L.INVALID_PROBLEM and append(qs=4094) == L.INVALID_PROBLEM
    assert append(act=F16, cache=F16, ks=1028) == L.INVALID_PROBLEM
    assert append(q=A, q_out=A, qs=6144) == L.INVALID_PROBLEM     # in place, but the rows lie apart
    assert append(k_out=A, ks=6144) == L.INVALID_PROBLEM


def test_decode_refusals():
    assert decode(seqs=0) == L.OK and decode(seqs=0, q=None, ws=None, ws_bytes=0) == L.OK
    for name in ("q", "kc", "vc", "out", "table", "lens"):
        assert decode(**{name: None}) == L.INVALID_PROBLEM, name
    for name in ("q", "kc", "vc", "out", "ws"):
        assert decode(**{name: A + 4}) == L.MISALIGNED, name
    assert decode(qs=4095) == L.INVALID_PROBLEM and decode(qs=4098) == L.INVALID_PROBLEM
    need = L.lib.fuelq_paged_attn_workspace_bytes(4, 32, 8, 128)
    if need:
        assert decode(ws=None) == L.WORKSPACE and decode(ws_bytes=need - 1) == L.WORKSPACE
    for bad in ((0, 32, 8, 128), (4, 30, 8, 128), (4, 32, 0, 128), (4, 32, 8, 96)):
        assert L.lib.fuelq_paged_attn_workspace_bytes(*bad) == 0


def test_prompt_refusals():
    assert prompt(seqs=0) == L.OK and prompt(rows=0, q=None) == L.OK
    assert prompt(act=Q4K) == L.NOT_SUPPORTED and prompt(hd=96) == L.NOT_SUPPORTED
    assert prompt(heads=30) == L.INVALID_PROBLEM and prompt(kv=0) == L.INVALID_PROBLEM
    assert prompt(seqs=-1) == L.INVALID_PROBLEM and prompt(rows=-1) == L.INVALID_PROBLEM and prompt(rows=1 << 31) == L.INVALID_PROBLEM
    assert prompt(seqs=(1 << 21) + 1) == L.NOT_SUPPORTED and prompt(rows=(1 << 30) - 255) == L.INVALID_PROBLEM
    assert prompt(heads=16384, kv=8, qs=16384 * 128) == L.INVALID_PROBLEM and decode(heads=16384, kv=8, qs=16384 * 128) == L.INVALID_PROBLEM
    for name in ("q", "k", "v", "out", "cu"):
        assert prompt(**{name: None}) == L.INVALID_PROBLEM, name
    for name in ("q", "k", "v", "out", "ws"):
        assert prompt(**{name: A + 8}) == L.MISALIGNED, name
    assert prompt(qs=4000) == L.INVALID_PROBLEM and prompt(ks=1026) == L.INVALID_PROBLEM and prompt(vs=1020) == L.INVALID_PROBLEM
    need = L.lib.fuelq_prompt_attn_workspace_bytes(F32, 64, 32, 8, 128)
    if need:
        assert prompt(ws=None) == L.WORKSPACE and prompt(ws_bytes=need - 1) == L.WORKSPACE


@pytest.mark.parametrize("call", [decode, prompt])
def test_scales(call):
    """Masked scores are -inf times the scale: it has to be a positive number."""
    for scale in (0.0, -0.1, float("inf"), float("nan")):
        assert call(scale=scale) == L.INVALID_PROBLEM


def test_there_is_no_cpu_path():
    q, kv, cache = torch.zeros(2, 4, 64), torch.zeros(2, 2, 64), torch.zeros(3, 2, 16, 64)
    ints, table, rope = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(8, 64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_append(kv, kv, cache, cache, table, ints, rope, rope, q=q)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attn_decode(q, cache, cache, table, ints)
    with pytest.raises(ValueError, match="CUDA"):
        ops.prompt_attn(q, kv, kv, ints)
