"""CPU tests of the exact path's operators: refusals, the frequency schedules, and the parameter blocks' layout.
No kernel is launched."""

from __future__ import annotations

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

import smaq_amd as S
from smaq_amd import _native

HEADER = (Path(__file__).resolve().parents[1] / "include" / "smaq_hip.h").read_text()


@pytest.mark.parametrize("name,mirror", [("smaq_rotary_params", _native.RotaryParams),
                                         ("smaq_packed_params", _native.PackedParams),
                                         ("smaq_paged_params", _native.PagedParams)])
def test_parameter_blocks_mirror_the_header(name, mirror):
    body = HEADER[HEADER.index(f"typedef struct {name} {{"):HEADER.index(f"}} {name};")]
    body = re.sub(r"/\*.*?\*/", "", body.split("{", 1)[1], flags=re.S)
    fields = []
    for decl in filter(None, (" ".join(d.split()) for d in body.split(";"))):
        base, names = re.match(r"((?:const )?(?:long long|int|float|double|void))\s*(.*)", decl).groups()
        first_ptr = names.startswith("*")
        for n in names.split(","):
            n = n.strip()
            assert n.startswith("*") == first_ptr or "*" not in names, decl
            kind = "ptr" if n.startswith("*") else {"long long": "ll", "int": "int", "float": "float"}[base]
            fields.append((n.lstrip("*").strip(), kind))
    kinds = {ctypes.c_int: "int", ctypes.c_float: "float", ctypes.c_longlong: "ll", ctypes.c_void_p: "ptr"}
    assert [(n, kinds[t]) for n, t in mirror._fields_] == fields


# ------------------------------------------------------------- frequencies ---

def test_frequencies_of_every_scaling():
    r, base, s, L = 64, 10000.0, 8.0, 4096
    f = [base ** (-2 * i / r) for i in range(r // 2)]
    plain = S.RotaryPositions(r, device="cpu")
    assert plain.freqs.dtype == torch.float64 and plain.gain == 1.0
    assert torch.allclose(plain.freqs, torch.tensor(f, dtype=torch.float64), rtol=1e-14)
    lin = S.RotaryPositions(r, scaling="linear", factor=s, device="cpu")
    assert torch.allclose(lin.freqs, plain.freqs / s, rtol=1e-14)
    ntk = S.RotaryPositions(r, scaling="ntk", factor=s, device="cpu")
    assert ntk.freqs[0] == 1.0 and math.isclose(float(ntk.freqs[-1]), f[-1] / s, rel_tol=1e-12)
    yarn = S.RotaryPositions(r, scaling="yarn", factor=s, original_length=L, device="cpu")
    ratio = yarn.freqs / plain.freqs
    turns = plain.freqs * L / (2 * math.pi)
    assert bool((ratio[turns > 64] == 1).all()) and torch.allclose(ratio[turns < 0.5], torch.tensor(1 / s).double())
    assert bool((ratio.diff() <= 1e-12).all()) and math.isclose(yarn.gain, 0.1 * math.log(s) + 1)
    own = S.RotaryPositions(r, freqs=[2.0] * 32, attention_factor=3.0, device="cpu")
    assert own.gain == 3.0 and bool((own.freqs == 2).all()) and own.to("cpu").rotary_dim == r
    assert S.RotaryPositions(0, device="cpu").freqs.numel() == 0


@pytest.mark.parametrize("kw", [dict(rotary_dim=63), dict(rotary_dim=-2), dict(rotary_dim=64, scaling="other"),
                                dict(rotary_dim=64, base=1.0), dict(rotary_dim=64, base=float("nan")),
                                dict(rotary_dim=64, scaling="linear", factor=0.5),
                                dict(rotary_dim=64, scaling="yarn", factor=2.0),
                                dict(rotary_dim=64, scaling="yarn", factor=2.0, original_length=64, beta_slow=40.0),
                                dict(rotary_dim=64, freqs=[1.0]), dict(rotary_dim=2, freqs=[1.0], scaling="ntk"),
                                dict(rotary_dim=2, freqs=[float("inf")]),
                                dict(rotary_dim=64, attention_factor=float("nan"))])
def test_rotary_positions_refusals(kw):
    with pytest.raises(ValueError):
        S.RotaryPositions(device="cpu", **kw)


# ---------------------------------------------------------------- refusals ---

def test_cpu_tensors_are_refused():
    x, i = torch.zeros(2, 2, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP kernels"):
        S.apply_norm_rotary(x, x, i, S.RotaryPositions(64, device="cpu"))
    with pytest.raises(ValueError, match="HIP kernels"):
        S.build_page_step(i, i, torch.zeros(2, 2, dtype=torch.int32), i, 16, 2)
    with pytest.raises(ValueError, match="HIP kernels"):
        S.compute_packed_attention(x, x, x, i)
    with pytest.raises(ValueError, match="HIP kernels"):
        S.compute_paged_attention(x, x[None], x[None], i[:, None], i, 4)


@pytest.fixture
def no_gpu_check(monkeypatch):
    """The checks of arguments behind the device check, on CPU tensors; no call gets as far as a launch."""
    check = _native.require_inputs
    monkeypatch.setattr(_native, "require_gpu", lambda *t: torch.device("cuda", 0))
    monkeypatch.setattr(_native, "require_inputs", lambda *a: (check(*a), 0)[1])

    def launch(*a, **k):
        raise AssertionError("launched")
    monkeypatch.setattr(_native, "launch_on", launch)


def _rotary_args(**kw):
    a = dict(q=torch.zeros(3, 4, 64), k=torch.zeros(3, 2, 64), positions=torch.zeros(3, dtype=torch.int64),
             rotary=S.RotaryPositions(64, device="cpu"))
    return {**a, **kw}


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(64)), dict(k=torch.zeros(4, 2, 64)), dict(k=torch.zeros(3, 2, 32)),
    dict(k=torch.zeros(3, 2, 64, dtype=torch.float16)), dict(positions=torch.zeros(2, dtype=torch.int64)),
    dict(positions=torch.zeros(3)), dict(positions=torch.zeros(3, dtype=torch.int16)), dict(q_weight=torch.ones(32)),
    dict(q_weight=torch.ones(64), k_weight=torch.ones(64, dtype=torch.float16)), dict(eps=-1.0),
    dict(eps=float("nan")), dict(weight_offset=float("inf")),
    dict(q=torch.zeros(3, 4, 64, dtype=torch.float64), k=None), dict(q=torch.zeros(3, 4, 64, requires_grad=True)),
    dict(q_weight=torch.ones(64, requires_grad=True))])
def test_norm_rotary_refusals(no_gpu_check, kw):
    with pytest.raises(ValueError):
        S.apply_norm_rotary(**_rotary_args(**kw))


def _page_args(**kw):
    a = dict(context_lens=torch.zeros(2, dtype=torch.int32), new_lens=torch.ones(2, dtype=torch.int32),
             block_table=torch.zeros(2, 4, dtype=torch.int32), free_blocks=torch.arange(8, dtype=torch.int32),
             block_size=16, num_tokens=2)
    return {**a, **kw}


@pytest.mark.parametrize("kw", [
    dict(context_lens=torch.zeros(2)), dict(context_lens=torch.zeros(3, dtype=torch.int32)),
    dict(new_lens=torch.zeros(1, 2, dtype=torch.int32)), dict(block_table=torch.zeros(2, 4, dtype=torch.int64)),
    dict(block_table=torch.zeros(1, 4, dtype=torch.int32)), dict(block_table=torch.zeros(4, 2, dtype=torch.int32).T),
    dict(free_blocks=torch.arange(8)), dict(free_blocks=torch.zeros(2, 2, dtype=torch.int32)), dict(num_tokens=-1)])
def test_page_step_refusals(no_gpu_check, kw):
    with pytest.raises(ValueError):
        S.build_page_step(**_page_args(**kw))


def test_page_step_refuses_a_table_that_shares_memory(no_gpu_check):
    buf = torch.zeros(20, dtype=torch.int32)
    for what, part in (("free_blocks", buf[4:12]), ("context_lens", buf[7:9])):
        with pytest.raises(ValueError, match="shares memory"):
            S.build_page_step(**_page_args(block_table=buf[:8].view(2, 4), **{what: part}))


H = torch.float16


def _packed_args(**kw):
    a = dict(q=torch.zeros(6, 4, 64, dtype=H), k=torch.zeros(6, 2, 64, dtype=H), v=torch.zeros(6, 2, 64, dtype=H),
             cu_seqlens=torch.tensor([0, 6], dtype=torch.int32))
    return {**a, **kw}


_PACKED_BAD = [
    dict(q=torch.zeros(6, 4, 64)), dict(q=torch.zeros(5, 4, 64, dtype=H)), dict(v=torch.zeros(6, 1, 64, dtype=H)),
    dict(k=torch.zeros(6, 2, 64, dtype=torch.bfloat16)), dict(q=torch.zeros(6, 3, 64, dtype=H)),
    dict(cu_seqlens=torch.zeros(0, dtype=torch.int32)), dict(cu_seqlens=torch.zeros(2)),
    dict(prefix_lens=torch.zeros(2, dtype=torch.int32)), dict(prefix_lens=torch.zeros(1)), dict(window=-1),
    dict(score_cap=-1.0), dict(score_cap=float("nan")), dict(score_cap=float("inf")), dict(scale=float("nan")),
    dict(alibi_slopes=torch.zeros(2)), dict(alibi_slopes=torch.zeros(4, dtype=torch.int32)),
    dict(out=torch.zeros(6, 4, 64)), dict(out=torch.zeros(6, 64, 4, dtype=H).transpose(1, 2)),
    dict(q=torch.zeros(6, 4, 64, dtype=H, requires_grad=True))]


@pytest.mark.parametrize("kw", _PACKED_BAD)
def test_packed_attention_refusals(no_gpu_check, kw):
    with pytest.raises(ValueError):
        S.compute_packed_attention(**_packed_args(**kw))


@pytest.mark.parametrize("D", [4, 60, 264])
def test_packed_attention_refuses_head_dims(no_gpu_check, D):
    x = torch.zeros(6, 2, D, dtype=H)
    with pytest.raises(ValueError, match="head_dim"):
        S.compute_packed_attention(x, x, x, torch.tensor([0, 6]))


def test_out_must_not_share_memory(no_gpu_check):
    buf = torch.zeros(6 * 4 * 64 + 64, dtype=H)
    q = buf[:6 * 4 * 64].view(6, 4, 64)
    with pytest.raises(ValueError, match="shares memory"):
        S.compute_packed_attention(**_packed_args(q=q, out=q))
    with pytest.raises(ValueError, match="shares memory"):
        S.compute_paged_attention(**_paged_args(q=q[:3], out=q[1:4]))


def _paged_args(**kw):
    a = dict(q=torch.zeros(3, 4, 64, dtype=H), k_cache=torch.zeros(5, 16, 2, 64, dtype=H),
             v_cache=torch.zeros(5, 16, 2, 64, dtype=H), block_table=torch.zeros(3, 2, dtype=torch.int32),
             seq_lens=torch.ones(3, dtype=torch.int32), max_seq_len=32)
    return {**a, **kw}


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(3, 4, 64)), dict(q=torch.zeros(3, 3, 64, dtype=H)), dict(q=torch.zeros(3, 4, 32, dtype=H)),
    dict(v_cache=torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16)), dict(v_cache=torch.zeros(4, 16, 2, 64, dtype=H)),
    dict(k_cache=torch.zeros(5, 8, 2, 64, dtype=H), v_cache=torch.zeros(5, 8, 2, 64, dtype=H)),
    dict(k_cache=torch.zeros(5, 16, 2, 65, dtype=H)[..., :64]), dict(block_table=torch.zeros(2, 2, dtype=torch.int32)),
    dict(block_table=torch.zeros(3, 2)), dict(seq_lens=torch.ones(2, dtype=torch.int32)), dict(seq_lens=torch.ones(3)),
    dict(max_seq_len=-1), dict(window=-3), dict(score_cap=float("inf")), dict(scale=float("inf")),
    dict(alibi_slopes=torch.zeros(3)), dict(out=torch.zeros(3, 4, 64)),
    dict(q=torch.zeros(3, 4, 64, dtype=H, requires_grad=True))])
def test_paged_attention_refusals(no_gpu_check, kw):
    with pytest.raises(ValueError):
        S.compute_paged_attention(**_paged_args(**kw))


def test_c_entries_refuse_before_any_launch():
    lib, d = _native.lib(), 4096
    p = _native.RotaryParams()
    assert lib.smaq_norm_rotary(None, None) == -1
    p.tokens, p.n_q_heads, p.head_dim, p.rotary_dim = 1, 1, 64, 63
    assert lib.smaq_norm_rotary(ctypes.byref(p), None) == -1 and b"rotary_dim 63" in lib.smaq_last_error()
    p.rotary_dim, p.dtype = 64, 9
    assert lib.smaq_norm_rotary(ctypes.byref(p), None) == -2
    p.dtype = 0
    assert lib.smaq_norm_rotary(ctypes.byref(p), None) == -1 and b"null pointer" in lib.smaq_last_error()
    p.tokens = 0
    assert lib.smaq_norm_rotary(ctypes.byref(p), None) == 0
    c = ctypes.c_void_p(d)
    assert lib.smaq_page_step(c, 4, c, 4, 8001, c, 4, c, 4, 16, 4, c, c, c, c, c, None) == -1
    assert lib.smaq_page_step(c, 2, c, 4, 1, c, 4, c, 4, 16, 4, c, c, c, c, c, None) == -1
    assert lib.smaq_page_step(c, 4, c, 4, 1, c, 4, c, 4, 0, 4, c, c, c, c, c, None) == -1
    assert lib.smaq_page_step(c, 4, c, 4, 1, None, 4, c, 4, 16, 4, c, c, c, c, c, None) == -1
    k = _native.PackedParams()
    assert lib.smaq_packed_attention(None, None) == -1
    k.dtype, k.n_docs, k.n_tokens, k.n_q_heads, k.n_kv_heads, k.head_dim = 1, 1, 4, 4, 3, 64
    assert lib.smaq_packed_attention(ctypes.byref(k), None) == -1
    k.n_kv_heads, k.head_dim = 2, 60
    assert lib.smaq_packed_attention(ctypes.byref(k), None) == -1 and b"head_dim 60" in lib.smaq_last_error()
    k.head_dim, k.dtype = 64, 0
    assert lib.smaq_packed_attention(ctypes.byref(k), None) == -2
    k.dtype = 1
    assert lib.smaq_packed_attention(ctypes.byref(k), None) == -1 and b"null pointer" in lib.smaq_last_error()
    k.q = k.k = k.v = k.out = k.starts = d
    k.q_stride_t = 12
    assert lib.smaq_packed_attention(ctypes.byref(k), None) == -1 and b"16 bytes" in lib.smaq_last_error()
    k.q_stride_t, k.v = 0, d + 2
    assert lib.smaq_packed_attention(ctypes.byref(k), None) == -1 and b"16 bytes" in lib.smaq_last_error()
    g = _native.PagedParams()
    assert lib.smaq_paged_attention(None, None) == -1 and lib.smaq_paged_workspace_bytes(None) == -1
    g.dtype, g.batch, g.n_q_heads, g.n_kv_heads, g.head_dim, g.block_size = 1, 2, 4, 2, 64, 24
    assert lib.smaq_paged_attention(ctypes.byref(g), None) == -1 and b"block_size 24" in lib.smaq_last_error()
    g.block_size, g.max_seq_len, g.max_blocks, g.num_blocks = 16, 64, 4, 4
    assert lib.smaq_paged_attention(ctypes.byref(g), None) == -1 and b"null pointer" in lib.smaq_last_error()
    g.q = g.out = g.seq_lens = g.block_table = g.k_cache = g.v_cache = d
    g.k_stride_t = 4
    assert lib.smaq_paged_attention(ctypes.byref(g), None) == -1 and b"16 bytes" in lib.smaq_last_error()


@pytest.mark.parametrize("kw", [dict(scale=1e39), dict(scale=-1e38), dict(score_cap=1e-50), dict(score_cap=1e30)])
def test_scales_and_caps_beyond_fp32_are_refused(no_gpu_check, kw):
    with pytest.raises(ValueError, match="scale|score_cap"):
        S.compute_packed_attention(**_packed_args(**kw))
    with pytest.raises(ValueError, match="scale|score_cap"):
        S.compute_paged_attention(**_paged_args(**kw))
    k, g = _native.PackedParams(), _native.PagedParams()
    for p, fn in ((k, "smaq_packed_attention"), (g, "smaq_paged_attention")):
        p.dtype, p.n_q_heads, p.n_kv_heads, p.head_dim = 1, 2, 2, 64
        p.scale, p.score_cap = kw.get("scale", 1.0), kw.get("score_cap", 0.0)
        if p is g:
            p.block_size = 16
        if kw.get("score_cap") != 1e-50:  # which a float argument turns into none
            assert getattr(_native.lib(), fn)(ctypes.byref(p), None) == -1 and b"scale" in _native.lib().smaq_last_error()


@pytest.mark.parametrize("kw", [dict(eps=1e39), dict(weight_offset=-1e39)])
def test_norm_constants_beyond_fp32_are_refused(no_gpu_check, kw):
    with pytest.raises(ValueError):
        S.apply_norm_rotary(**_rotary_args(**kw))
    with pytest.raises(ValueError):
        S.RotaryPositions(64, attention_factor=1e39, device="cpu")


@pytest.mark.parametrize("kw", [dict(block_size=0), dict(block_size=2 ** 32 + 16), dict(num_tokens=2 ** 31)])
def test_page_sizes_beyond_an_int_are_refused(no_gpu_check, kw):
    with pytest.raises(ValueError, match="block_size"):
        S.build_page_step(**_page_args(**kw))
