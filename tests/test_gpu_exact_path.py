"""GPU tests of the exact path's operators against plain statements in 64 bits.

Tolerances.  Half a step of the output type is u (bf16 2^-8, fp16 2^-11, fp32
2^-24, relative).  The rotary pass computes in fp32: a mean of D squares and its
root cost less than (D/2 + 4) 2^-24 relative, weights, gain, sine and cosine and
the rotation a dozen more roundings of the pair's magnitude, so
u |y| + (D/2 + 16) 2^-24 (|a| + |b|).  Attention: see ``_bound``.
"""

from __future__ import annotations

import math

import pytest
import torch

import smaq_amd as S

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
INF = float("inf")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------ rotary ---

def _rotary_oracle(x, positions, rot, w, eps, w0):
    """(y, magnitude of the rotated pair per element) in 64 bits."""
    y = x.double()
    if w is not None:
        y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps) * (w.double() + w0)
    r, out, mag = rot.rotary_dim, y.clone(), y.abs().clone()
    i = torch.arange(r // 2, device=x.device)
    ia, ib = (2 * i, 2 * i + 1) if rot.interleaved else (i, r // 2 + i)
    ang = positions.double()[..., None, None] * rot.freqs
    c, s = ang.cos() * rot.gain, ang.sin() * rot.gain
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * rot.gain
    return out, mag


def _check_rotary(got, x, positions, rot, w, eps=1e-6, w0=0.0):
    ref, mag = _rotary_oracle(x, positions, rot, w, eps, w0)
    tol = HALF_STEP[x.dtype] * ref.abs() + (x.shape[-1] / 2 + 16) * 2.0 ** -24 * mag
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25   # half a step below fp16's normal range
    assert got.dtype == x.dtype and got.shape == x.shape and got.is_contiguous()
    bad = (got.double() - ref).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} beyond, worst {float((got.double() - ref).abs().max())}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,r,interleaved", [(128, 128, False), (128, 64, True), (64, 64, False), (256, 128, False),
                                             (256, 256, True), (96, 96, False), (80, 32, True), (128, 24, False),
                                             (10, 6, False), (7, 2, True), (1, 0, False), (1024, 1024, False)])
def test_norm_rotary(dev, dtype, D, r, interleaved):
    g = _gen(D + r)
    rot = S.RotaryPositions(r, interleaved=interleaved)
    for T, hq, hk in ((1, 1, 1), (5, 7, 1), (67, 28, 4), (130, 3, 3)):
        if T * D > 40000:
            continue
        q = (3 * torch.randn(T, hq, D, generator=g, device=dev)).to(dtype)
        k = torch.randn(T, hk, D, generator=g, device=dev).to(dtype)
        w = (1 + 0.3 * torch.randn(2, D, generator=g, device=dev)).to(dtype)
        pos = torch.randint(0, 1 << 20, (T,), generator=g, device=dev)
        a, b = S.apply_norm_rotary(q, k, pos, rot, q_weight=w[0], k_weight=w[1])
        _check_rotary(a, q, pos, rot, w[0])
        _check_rotary(b, k, pos, rot, w[1])
        a, b = S.apply_norm_rotary(q, k, pos.int(), rot, k_weight=w[1].float(), eps=0.1, weight_offset=1.0)
        _check_rotary(a, q, pos, rot, None)
        _check_rotary(b, k, pos, rot, w[1].float(), 0.1, 1.0)


@pytest.mark.parametrize("kw", [dict(scaling="linear", factor=8.0), dict(scaling="ntk", factor=8.0),
                                dict(scaling="yarn", factor=32.0, original_length=4096),
                                dict(freqs=[0.5 ** i for i in range(64)], attention_factor=0.7)])
def test_norm_rotary_scalings_at_far_positions(dev, kw):
    g = _gen(5)
    rot = S.RotaryPositions(128, **kw)
    q = torch.randn(9, 4, 128, generator=g, device=dev)
    pos = torch.tensor([0, 1, -1, 4095, 131071, 1048575, 2 ** 31 - 1, 2 ** 31, -(2 ** 33)], device=dev)
    a, none = S.apply_norm_rotary(q, None, pos, rot)
    assert none is None
    # 64-bit angles: an angle of 2^33 turns has an error of 2^-20, which the oracle shares in part
    _check_rotary(a[:-1], q[:-1], pos[:-1], rot, None)
    assert bool(torch.isfinite(a).all())


def test_norm_rotary_reads_views_in_place(dev):
    """Views of a packed projection, an odd element offset, transposed tokens, and 4-D inputs."""
    g = _gen(6)
    rot = S.RotaryPositions(64)
    w = torch.rand(64, generator=g, device=dev).bfloat16()
    buf = torch.randn(33 * 6 * 64 + 3, generator=g, device=dev).bfloat16()
    pos = torch.arange(33, device=dev) * 7
    for off in (0, 1, 3):
        qkv = buf[off:off + 33 * 6 * 64].view(33, 6, 64)
        q, k = qkv[:, :4], qkv[:, 4:5]
        a, b = S.apply_norm_rotary(q, k, pos, rot, w, w)
        _check_rotary(a, q, pos, rot, w)
        _check_rotary(b, k, pos, rot, w)
    q = buf[:32 * 64 * 3].view(3, 64, 32).transpose(1, 2)[..., :64].transpose(0, 1)   # strided last dim
    a, _ = S.apply_norm_rotary(q, None, pos[:32], rot)
    _check_rotary(a, q, pos[:32], rot, None)
    x = torch.randn(2, 5, 3, 64, generator=g, device=dev).half()
    p4 = torch.arange(10, device=dev).view(2, 5)
    a, b = S.apply_norm_rotary(x, x[..., :2, :], p4, rot)
    _check_rotary(a, x, p4, rot, None)
    _check_rotary(b, x[..., :2, :], p4, rot, None)
    for T, hk in ((0, 2), (3, 0)):
        a, b = S.apply_norm_rotary(x.view(10, 3, 64)[:T], x.view(10, 3, 64)[:T, :hk], p4.view(-1)[:T], rot)
        assert a.shape == (T, 3, 64) and b.shape == (T, hk, 64)
    _check_rotary(a, x.view(10, 3, 64)[:3], p4.view(-1)[:3], rot, None)


@pytest.mark.parametrize("dtype,interleaved", [(torch.bfloat16, False), (torch.float16, True), (torch.float32, False)])
def test_norm_rotary_of_a_long_prompt(dev, dtype, interleaved):
    """Results beyond what the caches hold take another kind of store."""
    T = 7001 if dtype == torch.float32 else 14001
    x = torch.randn(T, 20, 128, generator=_gen(8), device=dev).to(dtype)
    rot, pos = S.RotaryPositions(64, interleaved=interleaved), torch.arange(T, device=dev)
    w = torch.rand(128, generator=_gen(9), device=dev).to(dtype)
    a, b = S.apply_norm_rotary(x, x[:, :3], pos, rot, w, w)
    _check_rotary(a, x, pos, rot, w)
    _check_rotary(b, x[:, :3], pos, rot, w)


def test_norm_rotary_keeps_nonfinite_values_in_their_row(dev):
    g = _gen(7)
    rot = S.RotaryPositions(128)
    q = torch.randn(4, 3, 128, generator=g, device=dev).bfloat16()
    pos = torch.arange(4, device=dev)
    w = torch.ones(128, device=dev).bfloat16()
    clean, _ = S.apply_norm_rotary(q, None, pos, rot, w)
    bad = q.clone()
    bad[2, 1, 5] = float("nan")
    bad[3, 0, 0] = INF
    got, _ = S.apply_norm_rotary(bad, None, pos, rot, w)
    assert bool(torch.isnan(got[2, 1]).all()) and bool(torch.isnan(got[3, 0, 0]))
    keep = torch.ones(4, 3, dtype=torch.bool, device=dev)
    keep[2, 1] = keep[3, 0] = False
    assert torch.equal(got[keep], clean[keep])
    zero, _ = S.apply_norm_rotary(torch.zeros_like(q), None, pos, rot, w)
    assert bool((zero == 0).all())


# ------------------------------------------------------------------- pages ---

def _pages_oracle(ctx, new, table, free, bs, tokens):
    table, free = table.tolist(), free.tolist()
    width = len(table[0]) if table else 0
    e, slots, positions, starts, total, unplaced = 0, [], [], [0], 0, 0
    for b, (c, m) in enumerate(zip(ctx, new)):
        c, m = max(c, 0), max(m, 0)
        for col in range(-(-c // bs), -(-(c + m) // bs)):
            if col < width:
                table[b][col] = free[e] if e < len(free) else -1
            e += 1
        for p in range(c, c + m):
            blk = table[b][p // bs] if p // bs < width else -1
            if len(slots) < tokens:
                slots.append(blk * bs + p % bs if blk >= 0 else -1)
                positions.append(p)
                unplaced += blk < 0
            else:
                unplaced += 1
        total += m
        starts.append(total)
    pad = tokens - len(slots)
    return (table, slots + [-1] * pad, positions + [0] * pad, starts, [max(c, 0) + max(m, 0) for c, m in zip(ctx, new)],
            [e, unplaced])


def _pages_case(ctx, new, bs, width, n_free, tokens, dev, holes=(), wide=False):
    g = torch.Generator().manual_seed(len(ctx) + bs)
    ids = torch.randperm(4 * len(ctx) * max(width, 1) + n_free + 8, generator=g).int()
    table = ids[:len(ctx) * width].view(len(ctx), width).clone()
    for b, col in holes:
        table[b, col] = -1
    free = ids[len(ctx) * width:len(ctx) * width + n_free].clone()
    want = _pages_oracle(ctx, new, table, free, bs, tokens)
    dt = torch.int64 if wide else torch.int32
    c, m, t, f = torch.tensor(ctx, dtype=dt).to(dev), torch.tensor(new, dtype=dt).to(dev), table.to(dev), free.to(dev)
    for _ in range(2):   # the same call again changes nothing
        step = S.build_page_step(c, m, t, f, bs, tokens)
        assert t.tolist() == want[0]
        for got, ref in zip(step, want[1:]):
            assert got.tolist() == list(ref)
    return step


def test_page_step_small(dev):
    _pages_case([], [], 16, 0, 0, 0, dev)
    _pages_case([], [], 16, 3, 2, 5, dev)
    _pages_case([0], [1], 16, 1, 1, 1, dev)
    _pages_case([5, 16, 0, 31, 32], [1, 1, 0, 1, 1], 16, 4, 8, 4, dev, wide=True)
    _pages_case([5, 16, 0, 31, 32], [40, 1, 17, 0, 100], 16, 9, 40, 200, dev)          # padded step
    _pages_case([5, 16, 0], [40, 20, 17], 16, 9, 40, 30, dev)                           # fewer rows than tokens
    _pages_case([5, 16, 0, 7], [40, 20, 17, 90], 16, 9, 5, 167, dev)                    # free list too short
    _pages_case([5, 16, 0, 7], [40, 20, 17, 90], 16, 3, 40, 167, dev)                   # rows too short
    _pages_case([5, 16, 50], [40, 20, 3], 16, 9, 40, 63, dev, holes=((0, 0), (2, 3)))    # no page behind the last token
    _pages_case([-3, 4], [6, -2], 16, 2, 4, 8, dev)                                      # negative lengths are 0
    _pages_case([3, 4], [6, 2], 16, 0, 4, 8, dev)
    _pages_case([3, 4], [6, 2], 1, 12, 10, 8, dev)
    _pages_case([10, 4], [6, 7], 7, 4, 3, 13, dev)


@pytest.mark.parametrize("n", [63, 64, 255, 256, 257, 1000, 8000])
def test_page_step_many_requests(dev, n):
    g = torch.Generator().manual_seed(n)
    ctx = torch.randint(0, 200, (n,), generator=g).tolist()
    new = torch.where(torch.rand(n, generator=g) < 0.1, torch.randint(0, 90, (n,), generator=g),
                      torch.ones(n, dtype=torch.int64)).tolist()
    _pages_case(ctx, new, 16, 19, sum(new) // 16 + n, sum(new) + 3, dev)


def test_page_step_saturates_and_refuses(dev):
    big = torch.tensor([2 ** 31 - 1, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    table = torch.zeros(2, 2, dtype=torch.int32, device=dev)
    step = S.build_page_step(big, big, table, torch.arange(4, dtype=torch.int32, device=dev), 16, 4)
    assert step.slot_mapping.tolist() == [-1] * 4 and step.seq_lens.tolist() == [2 ** 31 - 1] * 2
    assert step.query_start_loc.tolist() == [0, 2 ** 31 - 1, 2 ** 31 - 1] and step.status[1] == 2 ** 31 - 1
    many = torch.zeros(8001, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="8001 requests"):
        S.build_page_step(many, many, torch.zeros(8001, 1, dtype=torch.int32, device=dev), many, 16, 1)
    with pytest.raises(ValueError, match="block_size"):
        S.build_page_step(big, big, table, big, 0, 1)


# --------------------------------------------------------------- attention ---

def _scores64(q, k, i, j, scale, cap, slope):
    x = (q.double() @ k.double().T.contiguous()) * scale
    if cap:
        x = cap * torch.tanh(x / cap)
    if slope is not None:
        x = x - float(slope) * (i[:, None] - j[None, :]).abs().double()
    return x


def _bound(x, w, q, k, v, o, scale, cap, dtype):
    """Largest error of an output.  With A = sum w |v| and u half a step of the type:
    weights rounded to the type u A, the result u |o|; a score carries D products and
    sums of at most scale |q||k|, a few roundings of itself and of the cap
    (2^-21 of it; the distance bias is part of x), d = 2^-24 (D scale |q||k| + 8 |x| +
    8 cap), and moves a weight and the sum by as much: 2 d A, and e^(2 d) - 1 of it when
    d is not small; n sums n 2^-24 A.  fp16 weights below 2^-14 of the largest are off by
    2^-25 each: n 2^-25 max |v|."""
    n = k.shape[0]
    A = w @ v.double().abs()
    big = q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()
    seen = x.masked_fill(x == -INF, 0).abs().amax()
    d = 2.0 ** -24 * (q.shape[1] * abs(scale) * big + 8 * seen + 8 * cap)
    u = HALF_STEP[dtype]
    tol = (u + torch.expm1(2 * d) + n * 2.0 ** -24) * A + u * o.abs()
    if dtype == torch.float16:
        tol = tol + n * 2.0 ** -25 * v.double().abs().amax() + 2.0 ** -25
    return tol * (1 + 2.0 ** -6)   # products of the terms above


def _attend64(q, k, v, i, j, seen, scale, cap, slope, dtype):
    x = _scores64(q, k, i, j, scale, cap, slope).masked_fill(~seen, -INF)
    w = torch.softmax(x, -1)
    o = w @ v.double()
    return o, _bound(x, w, q, k, v, o, scale, cap, dtype)


def _close(got, ref, tol, what):
    err = (got.double() - ref).abs()
    assert not bool((~(err <= tol)).any()), f"{what}: worst error {float(err.max())} where {float(tol.flatten()[err.argmax()])} is allowed"


def _qkv(dev, T, hq, hkv, D, dtype, seed, gain=2.0):
    x = torch.randn(T, hq + 2 * hkv, D, generator=_gen(seed), device=dev)
    x[:, :hq] *= gain
    x = x.to(dtype)
    return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]


def _starts(lens, dev):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)


def _check_packed(dev, lens, hq, hkv, D, dtype, seed=1, causal=True, prefix=None, window=0, cap=0.0, slopes=None,
                  scale=None, heads=None, gain=2.0):
    q, k, v = _qkv(dev, sum(lens), hq, hkv, D, dtype, seed, gain)
    pl = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=dev)
    out = S.compute_packed_attention(q, k, v, _starts(lens, dev), scale=scale, causal=causal, prefix_lens=pl,
                                     window=window, score_cap=cap, alibi_slopes=slopes)
    scale = 1 / math.sqrt(D) if scale is None else scale
    t = 0
    for b, n in enumerate(lens):
        i = torch.arange(n, device=dev)
        seen = (i[None, :] <= i[:, None]) if causal else torch.ones(n, n, dtype=torch.bool, device=dev)
        if window:
            seen = seen & (i[None, :] > i[:, None] - window)
        if prefix is not None:
            seen = seen | (i[None, :] < prefix[b])
        for h in heads or range(hq):
            s = slice(t, t + n)
            if n:
                ref, tol = _attend64(q[s, h], k[s, h * hkv // hq], v[s, h * hkv // hq], i, i, seen, scale, cap,
                                     None if slopes is None else slopes[h], dtype)
                _close(out[s, h], ref, tol, f"document {b} head {h}")
        t += n
    return out


RAGGED = [1, 0, 63, 64, 65, 2, 127, 128, 129, 31, 33, 200, 255, 257, 16]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,D", [(4, 1, 128), (2, 2, 64), (2, 1, 256), (7, 1, 128), (2, 1, 96), (1, 1, 8), (3, 1, 200)])
def test_packed_ragged_documents(dev, dtype, hq, hkv, D):
    _check_packed(dev, RAGGED, hq, hkv, D, dtype)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kw", [dict(causal=False), dict(cap=50.0), dict(cap=3.0, causal=False), dict(cap=5000.0),
                                dict(window=1), dict(window=17), dict(window=64), dict(window=100, causal=False),
                                dict(window=2 ** 31 - 1), dict(alibi=True), dict(alibi=True, causal=False),
                                dict(prefix=True), dict(prefix=True, window=20), dict(prefix=True, alibi=True, cap=20.0),
                                dict(scale=0.0), dict(scale=-0.3), dict(gain=40.0)])
def test_packed_masks_caps_and_biases(dev, D, kw):
    kw = dict(kw)
    lens = [130, 1, 300, 64, 77]
    if kw.pop("alibi", False):
        kw["slopes"] = torch.tensor([0.5, 0.01], device=dev)
    if kw.pop("prefix", False):
        kw["prefix"] = [0, 1, 150, 64, 100]
    _check_packed(dev, lens, 2, 1, D, torch.bfloat16, seed=3, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_packed_long_documents(dev, dtype):
    _check_packed(dev, [2500, 700, 1800], 4, 1, 128, dtype, seed=4, heads=(0, 3))
    _check_packed(dev, [3001], 8, 8, 64, dtype, seed=5, cap=30.0, heads=(0, 5))


@pytest.mark.parametrize("lens", [[1] * 62, [1] * 63, [1] * 64, [2] * 100 + [0] * 80 + [130] + [1] * 50, [0] * 200 + [70],
                                  [300] + [0] * 70, [33, 0, 0, 31] * 30, [0] * 5000 + [3, 200, 1]])
def test_packed_many_documents(dev, lens):
    """Below and above the 63 documents whose starts one load holds, and runs of empty ones."""
    _check_packed(dev, lens, 2, 1, 128, torch.bfloat16, seed=21)
    _check_packed(dev, lens, 2, 2, 64, torch.float16, seed=22, window=9, prefix=[min(n, 5) for n in lens])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv,lens", [(8, 8, [500]), (4, 2, [1100, 900]), (8, 2, [2048]), (2, 1, [257]),
                                         (8, 8, [1000, 40, 1100])])
def test_packed_key_groups(dev, D, hq, hkv, lens):
    """Grids of a workgroup or two a CU, whose units have two groups of waves over the keys: causal and not, with a
    gap between prefix and window, and values that are not finite."""
    heads = (0, hq - 1)
    _check_packed(dev, lens, hq, hkv, D, torch.bfloat16, seed=23, heads=heads)
    _check_packed(dev, lens, hq, hkv, D, torch.float16, seed=24, causal=False, cap=30.0, heads=heads)
    _check_packed(dev, lens, hq, hkv, D, torch.bfloat16, seed=25, prefix=[50] * len(lens), window=70, heads=heads)
    q, k, v = _qkv(dev, sum(lens), hq, hkv, D, torch.bfloat16, 26)
    starts, at = _starts(lens, dev), lens[0] - 20
    clean = S.compute_packed_attention(q, k, v, starts)
    bad = v.clone()
    bad[at:lens[0]] = float("nan")
    got = S.compute_packed_attention(q, k, bad, starts)
    assert torch.equal(got[:at], clean[:at]) and torch.equal(got[lens[0]:], clean[lens[0]:])
    assert bool(torch.isnan(got[at:lens[0]]).all())


def test_packed_results_do_not_change_from_run_to_run(dev):
    q, k, v = _qkv(dev, 3000, 8, 2, 128, torch.bfloat16, 27)
    starts = _starts([1700, 1300], dev)
    ref = S.compute_packed_attention(q, k, v, starts, score_cap=50.0)
    for _ in range(3):
        assert torch.equal(S.compute_packed_attention(q, k, v, starts, score_cap=50.0), ref)


def test_packed_one_token(dev):
    q, k, v = _qkv(dev, 1, 4, 2, 128, torch.bfloat16, 6)
    out = S.compute_packed_attention(q, k, v, torch.tensor([0, 1], device=dev))
    assert torch.equal(out, v.repeat_interleave(2, 1))
    assert S.compute_packed_attention(q[:0], k[:0], v[:0], torch.tensor([0], device=dev)).shape == (0, 4, 128)


def test_packed_rows_of_no_document(dev):
    """A padded batch: rows behind the last document and before the first are zeros in a new result and untouched
    in a given one; starts beyond the rows are cut."""
    q, k, v = _qkv(dev, 300, 4, 2, 128, torch.float16, 7)
    starts = torch.tensor([5, 100, 100, 222], dtype=torch.int64, device=dev)
    new = S.compute_packed_attention(q, k, v, starts)
    assert bool((new[:5] == 0).all()) and bool((new[222:] == 0).all())
    out = torch.full_like(new, 7.0)
    assert S.compute_packed_attention(q, k, v, starts, out=out) is out
    assert bool((out[:5] == 7).all()) and bool((out[222:] == 7).all()) and torch.equal(out[5:222], new[5:222])
    none = S.compute_packed_attention(q, k, v, torch.tensor([0], dtype=torch.int32, device=dev))
    assert bool((none == 0).all())
    cut = S.compute_packed_attention(q, k, v, torch.tensor([-4, 100, 5000], dtype=torch.int32, device=dev))
    whole = S.compute_packed_attention(q, k, v, torch.tensor([0, 100, 300], dtype=torch.int32, device=dev))
    assert torch.equal(cut, whole)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), INF, -INF])
def test_packed_unseen_places_do_not_matter(dev, bad, D):
    """Row i of a causal document is the same whatever stands in rows above it, and rows of another document stay
    apart; rows that do see a NaN value are NaN."""
    lens, at = [70, 200, 90], 70 + 101
    q, k, v = _qkv(dev, 360, 2, 1, D, torch.bfloat16, 8)
    clean = S.compute_packed_attention(q, k, v, _starts(lens, dev))
    for which in "kv":
        x = {"k": k.clone(), "v": v.clone()}
        x[which][at:270] = bad
        got = S.compute_packed_attention(q, x["k"], x["v"], _starts(lens, dev))
        assert torch.equal(got[:at], clean[:at]) and torch.equal(got[270:], clean[270:])
        if which == "v":
            assert not bool(torch.isfinite(got[at:270]).any())
    x = v.clone()
    x[at, 0, 3] = bad
    got = S.compute_packed_attention(q, k, x, _starts(lens, dev), window=30)
    clean = S.compute_packed_attention(q, k, v, _starts(lens, dev), window=30)
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[at:at + 30, :, 3] = True
    assert torch.equal(got[~hit], clean[~hit]) and not bool(torch.isfinite(got[hit]).any())


def test_packed_infinite_scores(dev):
    """A score of -inf beside finite ones has no weight; a row of -inf alone is NaN, as its softmax."""
    q, k, v = (torch.ones(40, 1, 64, device=dev, dtype=torch.bfloat16) for _ in range(3))
    k[3] = -INF
    out = S.compute_packed_attention(q, k, v, torch.tensor([0, 40], device=dev))
    assert bool((out == 1).all())
    k[:] = -INF
    assert bool(torch.isnan(S.compute_packed_attention(q, k, v, torch.tensor([0, 40], device=dev))).all())
    capped = S.compute_packed_attention(q, k, v, torch.tensor([0, 40], device=dev), score_cap=10.0)
    assert bool((capped == 1).all())


def test_packed_and_rotary_offsets_beyond_32_bits(dev):
    """Rows that lie more than 2^31 elements into a packed projection."""
    T, hq, hkv, D, doc = 360000, 32, 8, 128, 48
    assert T * (hq + 2 * hkv) * D > 2 ** 31
    x = torch.empty(T, hq + 2 * hkv, D, dtype=torch.bfloat16, device=dev)
    x[:doc] = torch.randn(doc, hq + 2 * hkv, D, generator=_gen(28), device=dev)
    for i in range(doc, T, doc * 100):   # every document is the first one
        m = min(doc * 100, T - i)
        x[i:i + m] = x[:doc].repeat(100, 1, 1)[:m]
    starts = torch.arange(0, T + 1, doc, dtype=torch.int32, device=dev)
    out = S.compute_packed_attention(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], starts)
    assert bool(torch.isfinite(out[:doc]).all())
    q, k = S.apply_norm_rotary(x[:, :hq], x[:, hq:hq + hkv], torch.arange(T, device=dev) % doc, S.RotaryPositions(D))
    for t in (out, q, k):
        assert torch.equal(t.view(T // doc, doc, -1), t[:doc].reshape(1, doc, -1).expand(T // doc, -1, -1))


def test_packed_strides_and_alignment(dev):
    """Transposed, expanded and misaligned inputs give what contiguous ones give."""
    q, k, v = (t.contiguous() for t in _qkv(dev, 150, 4, 2, 64, torch.float16, 9))
    starts = _starts([100, 50], dev)
    ref = S.compute_packed_attention(q, k, v, starts)
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    kt = torch.zeros(150 * 2 * 64 + 1, dtype=torch.float16, device=dev)[1:].view(150, 2, 64).copy_(k)
    vt = torch.zeros(150, 2, 66, dtype=torch.float16, device=dev)[..., :64].copy_(v)
    vs = torch.zeros(150, 2, 64, 2, dtype=torch.float16, device=dev)[..., 0].copy_(v)
    for x in (vt, vs):
        assert torch.equal(S.compute_packed_attention(qt, kt, x, starts), ref)
    one = S.compute_packed_attention(q, k[:, :1].expand(150, 4, 64), v[:, :1].expand(150, 4, 64), starts)
    assert torch.equal(one, S.compute_packed_attention(q, k[:, :1], v[:, :1], starts))


# ------------------------------------------------------------------- paged ---

def _cache(dev, lens, bs, hkv, D, dtype, seed, spare=3):
    """A flash-layout cache whose other rows hold NaN, the pages of the sequences in shuffled order."""
    g = _gen(seed)
    held = [-(-n // bs) for n in lens]
    kv = torch.full((2, sum(held) + spare, bs, hkv, D), float("nan"), dtype=dtype, device=dev)
    perm = torch.randperm(sum(held) + spare, generator=g, device=dev).int()
    table = torch.full((len(lens), max(held + [1]) + 1), -1, dtype=torch.int32, device=dev)
    ks, vs, o = [], [], 0
    for b, n in enumerate(lens):
        table[b, :held[b]] = perm[o:o + held[b]]
        o += held[b]
        k, v = (torch.randn(n, hkv, D, generator=g, device=dev).to(dtype) for _ in range(2))
        j = torch.arange(n, device=dev)
        kv[0][table[b].long()[j // bs], j % bs] = k
        kv[1][table[b].long()[j // bs], j % bs] = v
        ks.append(k)
        vs.append(v)
    return kv, table, ks, vs


def _check_paged(dev, lens, hq, hkv, D, dtype, bs=16, seed=1, window=0, cap=0.0, slopes=None, bound=None, wide=False,
                 gain=2.0):
    kv, table, ks, vs = _cache(dev, lens, bs, hkv, D, dtype, seed)
    q = (gain * torch.randn(len(lens), hq, D, generator=_gen(seed + 50), device=dev)).to(dtype)
    sl = torch.tensor(lens, dtype=torch.int64 if wide else torch.int32, device=dev)
    out = S.compute_paged_attention(q, kv[0], kv[1], table, sl, bound or max(lens + [0]), window=window, score_cap=cap,
                                    alibi_slopes=slopes)
    for b, n in enumerate(lens):
        if n <= 0:
            assert bool((out[b] == 0).all())
            continue
        lo = max(0, n - window) if window else 0
        j = torch.arange(lo, n, device=dev)
        for h in range(hq):
            kh = h * hkv // hq
            ref, tol = _attend64(q[b, h:h + 1], ks[b][lo:, kh], vs[b][lo:, kh], j[-1:], j,
                                 torch.ones(1, n - lo, dtype=torch.bool, device=dev), 1 / math.sqrt(D), cap,
                                 None if slopes is None else slopes[h], dtype)
            _close(out[b, h:h + 1], ref, tol, f"sequence {b} head {h}")
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,D", [(8, 2, 128), (4, 4, 64), (4, 2, 256), (14, 2, 128), (6, 2, 96), (1, 1, 8),
                                      (32, 1, 128), (40, 2, 64), (3, 1, 200)])
def test_paged_ragged_sequences(dev, dtype, hq, hkv, D):
    _check_paged(dev, [1, 15, 16, 17, 0, 31, 32, 33, 100, 127, 128, 129, 300, 511, 513], hq, hkv, D, dtype)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kw", [dict(bs=32), dict(bs=48), dict(bs=256), dict(window=1), dict(window=20),
                                dict(window=128), dict(cap=50.0), dict(cap=2.0), dict(cap=5000.0), dict(alibi=True),
                                dict(alibi=True, window=77, cap=30.0), dict(wide=True), dict(bound=65536),
                                dict(gain=40.0)])
def test_paged_masks_caps_and_layouts(dev, D, kw):
    kw = dict(kw)
    if kw.pop("alibi", False):
        kw["slopes"] = torch.tensor([0.5, 0.01, 0.001, 1.0], device=dev)
    _check_paged(dev, [1, 700, 64, 350, 16], 4, 1, D, torch.bfloat16, seed=2, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_paged_long_sequences(dev, dtype):
    _check_paged(dev, [20011], 4, 1, 128, dtype, seed=3)
    _check_paged(dev, [9000, 5, 4096, 12345], 7, 1, 128, dtype, seed=4, cap=50.0)


@pytest.mark.parametrize("B", [63, 65, 300, 5000])
def test_paged_many_sequences(dev, B):
    """Shares that begin and end in any sequence, empty ones among them; every sequence has one page of its own, and a
    few have forty."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 17, (B,), generator=g)
    lens[torch.randint(0, B, (6,), generator=g)] = 640
    lens[0], lens[-1] = 0, 0
    bs, hkv, hq, D = 16, 4, 8, 64
    kv = torch.randn(2, B + 40, bs, hkv, D, generator=_gen(B), device=dev).half()
    table = torch.full((B, 40), -1, dtype=torch.int32)
    table[:, 0] = torch.arange(B)
    for b in (lens == 640).nonzero().flatten().tolist():
        table[b] = torch.randperm(B + 40, generator=g)[:40].int()
    q = torch.randn(B, hq, D, generator=_gen(B + 1), device=dev).half()
    out = S.compute_paged_attention(q, kv[0], kv[1], table.to(dev), lens.to(dev), 640)
    again = S.compute_paged_attention(q, kv[0], kv[1], table.to(dev), lens.to(dev).int(), 640)
    assert torch.equal(out, again)
    tab = table.to(dev).long()
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            assert bool((out[b] == 0).all())
            continue
        if B > 400 and n < 640 and b % 50:
            continue
        j = torch.arange(n, device=dev)
        for h in (0, hq - 1):
            k, v = (kv[i][tab[b][j // bs], j % bs, h * hkv // hq] for i in range(2))
            ref, tol = _attend64(q[b, h:h + 1], k, v, j[-1:], j, torch.ones(1, n, dtype=torch.bool, device=dev), 0.125, 0.0,
                                 None, torch.float16)
            _close(out[b, h:h + 1], ref, tol, f"sequence {b} head {h}")


@pytest.mark.parametrize("hq,hkv,D", [(16, 4, 128), (8, 8, 64), (80, 4, 128)])
def test_paged_heads_side_by_side(dev, hq, hkv, D):
    """Enough work that four heads are read together, sequences of all lengths, with and without a window."""
    lens = [4100, 1, 0, 2049, 3333, 16, 4096, 31, 1000, 2500] * 4
    for window in (0, 700):
        kv, table, ks, vs = _cache(dev, lens, 16, hkv, D, torch.bfloat16, 70)
        q = torch.randn(len(lens), hq, D, generator=_gen(71), device=dev).bfloat16()
        sl = torch.tensor(lens, device=dev)
        out = S.compute_paged_attention(q, kv[0], kv[1], table, sl, max(lens), window=window, score_cap=40.0)
        for b, n in enumerate(lens):
            lo = max(0, n - window) if window else 0
            j = torch.arange(lo, n, device=dev)
            for h in (0, hq // 2, hq - 1) if n else ():
                kh = h * hkv // hq
                ref, tol = _attend64(q[b, h:h + 1], ks[b][lo:, kh], vs[b][lo:, kh], j[-1:], j,
                                     torch.ones(1, n - lo, dtype=torch.bool, device=dev), 1 / math.sqrt(D), 40.0, None,
                                     torch.bfloat16)
                _close(out[b, h:h + 1], ref, tol, f"sequence {b} head {h}")
            if n == 0:
                assert bool((out[b] == 0).all())


def test_paged_scores_that_are_not_finite(dev):
    """A NaN key in one share makes its rows NaN, scores of -inf count for nothing beside finite ones, alone they are
    NaN; other sequences and heads keep their bits."""
    lens = [3000, 2000, 500]
    kv, table, ks, vs = _cache(dev, lens, 16, 2, 64, torch.float16, 72)
    q = torch.rand(3, 4, 64, generator=_gen(73), device=dev).half() + 0.1
    sl = torch.tensor(lens, device=dev)
    clean = S.compute_paged_attention(q, kv[0], kv[1], table, sl, 3000)
    page = int(table[0, 100])
    for bad, rows_nan in ((float("nan"), True), (-INF, False)):
        x = kv.clone()
        x[0, page, 3, 1] = bad
        got = S.compute_paged_attention(q, x[0], x[1], table, sl, 3000)
        assert torch.equal(got[1:], clean[1:]) and torch.equal(got[0, :2], clean[0, :2])
        assert bool(torch.isnan(got[0, 2:]).all()) == rows_nan and bool(torch.isfinite(got[0, 2:]).all()) != rows_nan
    x = kv.clone()
    x[0][:, :, 1] = -INF
    got = S.compute_paged_attention(q, x[0], x[1], table, sl, 3000)
    assert bool(torch.isnan(got[:, 2:]).all()) and torch.equal(got[:, :2], clean[:, :2])
    x = kv.clone()
    x[1, page, 3, 1, 5] = float("nan")
    got = S.compute_paged_attention(q, x[0], x[1], table, sl, 3000)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[0, 2:, 5] = True
    assert bool(torch.isnan(got[hit]).all()) and torch.equal(got[~hit], clean[~hit])


def test_paged_bad_pages_and_empty_sequences(dev):
    """Entries that are no block of the cache leave their tokens out; sequences of no token are zeros; lengths beyond
    the table or the bound are cut."""
    kv, table, ks, vs = _cache(dev, [100, 64, 40, 16], 16, 2, 64, torch.float16, 5)
    q = torch.randn(4, 4, 64, generator=_gen(6), device=dev).half()
    table[0, 2], table[0, 5], table[1, :] = -1, 2 ** 31 - 1, -7
    lens = torch.tensor([100, 64, -5, 16], dtype=torch.int32, device=dev)
    out = S.compute_paged_attention(q, kv[0], kv[1], table, lens, 100)
    assert bool((out[1] == 0).all()) and bool((out[2] == 0).all())
    j = torch.tensor([t for t in range(100) if t // 16 not in (2, 5)], device=dev)
    for h in range(4):
        ref, tol = _attend64(q[0, h:h + 1], ks[0][j, h // 2], vs[0][j, h // 2], j[-1:], j,
                             torch.ones(1, len(j), dtype=torch.bool, device=dev), 0.125, 0.0, None, torch.float16)
        _close(out[0, h:h + 1], ref, tol, f"head {h}")
    lens[3] = 10 ** 6                                     # 9 table entries, the last -1: 16 tokens are there
    wide = table.long()
    wide[0, 2], wide[0, 5], wide[1, :] = 2 ** 32, 2 ** 32 + 1, -(2 ** 40)       # no wrapping into the cache either
    assert torch.equal(S.compute_paged_attention(q, kv[0], kv[1], wide, lens.clamp(max=100), 100)[:3], out[:3])
    long = S.compute_paged_attention(q, kv[0], kv[1], table, lens, 10 ** 6)
    ok = S.compute_paged_attention(q, kv[0], kv[1], table, torch.tensor([100, 64, -5, 16], device=dev), 100)
    _close(long[3], ok[3].double(), 2 ** -10 * ok[3].double().abs() + 2 ** -10 * vs[3].abs().max().double(), "cut")
    assert bool((S.compute_paged_attention(q, kv[0], kv[1], table, lens, 0) == 0).all())
    assert bool((S.compute_paged_attention(q, kv[0][:0], kv[1][:0], table, lens, 100) == 0).all())
    assert bool((S.compute_paged_attention(q, kv[0], kv[1], table[:, :0], lens, 100) == 0).all())
    assert S.compute_paged_attention(q[:0], kv[0], kv[1], table, lens, 100).shape == (0, 4, 64)


def test_paged_other_cache_layouts(dev):
    """Head-major and interleaved key/value caches, a strided query, an int64 table and out=."""
    kv, table, _, _ = _cache(dev, [77, 130], 16, 2, 128, torch.bfloat16, 7)
    q = torch.randn(2, 4, 128, generator=_gen(8), device=dev).bfloat16()
    lens = torch.tensor([77, 130], device=dev)
    ref = S.compute_paged_attention(q, kv[0], kv[1], table, lens, 130)
    head_major = kv.transpose(2, 3).contiguous().transpose(2, 3)
    both = kv.transpose(0, 1).contiguous().transpose(0, 1)
    qs = torch.zeros(2, 4, 129, device=dev, dtype=torch.bfloat16)[..., :128].copy_(q)
    for c in (head_major, both):
        assert torch.equal(S.compute_paged_attention(qs, c[0], c[1], table.long(), lens, 130), ref)
    out = torch.empty_like(ref)
    assert S.compute_paged_attention(q, kv[0], kv[1], table, lens, 130, out=out) is out and torch.equal(out, ref)


def test_paged_offsets_beyond_32_bits(dev):
    """Pages whose rows lie more than 2^32 bytes, and 2^31 elements, into the cache."""
    bs, hkv, D = 16, 8, 128
    blocks = (1 << 31) // (bs * hkv * D) + 40
    kv = torch.empty(2, blocks, bs, hkv, D, dtype=torch.bfloat16, device=dev)
    n = 100
    last = torch.arange(blocks - 7, blocks, device=dev)
    k, v = (torch.randn(7 * bs, hkv, D, generator=_gen(9 + i), device=dev).bfloat16() for i in range(2))
    kv[0, blocks - 7:] = k.view(7, bs, hkv, D)
    kv[1, blocks - 7:] = v.view(7, bs, hkv, D)
    q = torch.randn(1, 8, D, generator=_gen(11), device=dev).bfloat16()
    far = S.compute_paged_attention(q, kv[0], kv[1], last[None], torch.tensor([n], device=dev), n)
    near = S.compute_paged_attention(q, kv[0, -7:], kv[1, -7:], torch.arange(7, device=dev)[None],
                                     torch.tensor([n], device=dev), n)
    assert torch.equal(far, near) and bool(torch.isfinite(far).all())


# ---------------------------------------------- streams, graphs, all of them ---

def test_operators_on_another_stream(dev):
    q, k, v = _qkv(dev, 400, 8, 2, 128, torch.bfloat16, 12)
    starts = _starts([250, 150], dev)
    kv, table, _, _ = _cache(dev, [500, 30], 16, 2, 128, torch.bfloat16, 13)
    lens, rot = torch.tensor([500, 30], device=dev), S.RotaryPositions(128)
    pos = torch.arange(400, device=dev)

    def all_of_them():
        a, b = S.apply_norm_rotary(q, k, pos, rot)
        return a, b, S.compute_packed_attention(a, b, v, starts), S.compute_paged_attention(a[:2], kv[0], kv[1], table,
                                                                                           lens, 500)
    ref = all_of_them()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_of_them()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, ref):
        assert torch.equal(a, b)


def test_graphs_replay_with_new_inputs(dev):
    """Two graphs of the serving step captured one after the other, replayed in turn with new lengths, beside eager
    calls: every replay is what the eager call gives."""
    bs, hq, hkv, D, B, width = 16, 8, 2, 128, 5, 40
    rot = S.RotaryPositions(D)
    w = torch.rand(D, generator=_gen(14), device=dev).bfloat16()
    qkv = torch.randn(B, hq + 2 * hkv, D, generator=_gen(15), device=dev).bfloat16()
    ctx = torch.tensor([0, 100, 5, 550, 33], dtype=torch.int32, device=dev)
    one = torch.ones(B, dtype=torch.int32, device=dev)
    table = torch.randperm(B * width, generator=_gen(16), device=dev).int().view(B, width)
    free = torch.arange(B * width, B * width + 8, dtype=torch.int32, device=dev)
    kv = torch.randn(2, B * width + 8, bs, hkv, D, generator=_gen(17), device=dev).bfloat16()

    def step():
        pages = S.build_page_step(ctx, one, table, free, bs, B)
        q, k = S.apply_norm_rotary(qkv[:, :hq], qkv[:, hq:hq + hkv], pages.positions, rot, w, w)
        kv[0].view(-1, hkv, D).index_copy_(0, pages.slot_mapping, k)
        kv[1].view(-1, hkv, D).index_copy_(0, pages.slot_mapping, qkv[:, hq + hkv:])
        return (S.compute_paged_attention(q, kv[0], kv[1], table, pages.seq_lens, width * bs, score_cap=50.0),
                S.compute_packed_attention(q, k, qkv[:, hq + hkv:], pages.query_start_loc), pages.slot_mapping)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for r in range(6):
        ctx.copy_(torch.tensor([r, 100 + 7 * r, 15 + r, 550 + r, 16 * r], dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, generator=_gen(20 + r), device=dev))
        want = [t.clone() for t in step()]
        graph, outs = graphs[r % 2]
        for t in outs:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), r


def test_a_prompt_and_its_decode_steps(dev):
    """The operators as a serving program runs them: pages, normed and rotated heads, a packed prefill, the tokens
    written through the slot map, and paged decode steps, against full attention over the same tokens."""
    bs, hq, hkv, D = 16, 8, 2, 64
    lens, steps = [37, 1, 130], 20
    total = [n + steps for n in lens]
    rot = S.RotaryPositions(D, scaling="yarn", factor=4.0, original_length=64)
    qw, kw = (1 + 0.1 * torch.randn(D, generator=_gen(30 + i), device=dev).half() for i in range(2))
    x = [torch.randn(n, hq + 2 * hkv, D, generator=_gen(40 + i), device=dev).half() for i, n in enumerate(total)]
    blocks = sum(-(-n // bs) for n in total)
    kv = torch.full((2, blocks, bs, hkv, D), float("nan"), dtype=torch.float16, device=dev)
    table = torch.full((3, -(-max(total) // bs)), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(blocks, generator=_gen(50), device=dev).int()
    held = torch.zeros(3, dtype=torch.int32, device=dev)
    outs = [[] for _ in lens]
    for s in range(steps + 1):
        new = lens if s == 0 else [1, 1, 1]
        at = [0, 0, 0] if s == 0 else [n + s - 1 for n in lens]
        qkv = torch.cat([t[a:a + m] for t, a, m in zip(x, at, new)])
        pages = S.build_page_step(held, torch.tensor(new, device=dev), table, free, bs, sum(new))
        taken, lost = pages.status.tolist()
        free, held = free[taken:], pages.seq_lens
        assert lost == 0
        q, k = S.apply_norm_rotary(qkv[:, :hq], qkv[:, hq:hq + hkv], pages.positions, rot, qw, kw)
        v = qkv[:, hq + hkv:]
        kv[0].view(-1, hkv, D)[pages.slot_mapping] = k
        kv[1].view(-1, hkv, D)[pages.slot_mapping] = v
        o = (S.compute_packed_attention(q, k, v, pages.query_start_loc, score_cap=30.0) if s == 0 else
             S.compute_paged_attention(q, kv[0], kv[1], table, pages.seq_lens, max(total), score_cap=30.0))
        for b, (i, j) in enumerate(zip(pages.query_start_loc.tolist(), pages.query_start_loc.tolist()[1:])):
            outs[b].append(o[i:j])
    assert free.numel() == 0
    for b, n in enumerate(total):
        pos = torch.arange(n, device=dev)
        q, k = S.apply_norm_rotary(x[b][:, :hq], x[b][:, hq:hq + hkv], pos, rot, qw, kw)
        got = torch.cat(outs[b])
        for h in range(hq):
            ref, tol = _attend64(q[:, h], k[:, h * hkv // hq], x[b][:, hq + hkv + h * hkv // hq], pos, pos,
                                 pos[None, :] <= pos[:, None], 1 / math.sqrt(D), 30.0, None, torch.float16)
            _close(got[:, h], ref, tol, f"request {b} head {h}")


def test_gradients_are_refused(dev):
    q, k, v = _qkv(dev, 4, 2, 1, 64, torch.float16, 60)
    starts = torch.tensor([0, 4], device=dev)
    with pytest.raises(ValueError, match="no gradients"):
        S.compute_packed_attention(q, k.clone().requires_grad_(), v, starts)
    with torch.no_grad():
        S.compute_packed_attention(q, k.clone().requires_grad_(), v, starts)


def test_two_calls_at_once(dev):
    """Two streams run the same operators on their own inputs side by side: each gets what it gets alone."""
    kv, table, _, _ = _cache(dev, [4000, 7, 2500], 16, 4, 128, torch.bfloat16, 40)
    rot = S.RotaryPositions(128)
    starts, pos = _starts([700, 333], dev), torch.arange(1033, device=dev)
    qkv = [_qkv(dev, 1033, 8, 4, 128, torch.bfloat16, 41 + i) for i in range(2)]
    lens = [torch.tensor(x, dtype=torch.int32, device=dev) for x in ([4000, 7, 2500], [1999, 0, 2500])]
    ctx = [torch.tensor(x, dtype=torch.int32, device=dev) for x in ([17, 3, 16], [0, 31, 5])]
    tables = [torch.zeros(3, 8, dtype=torch.int32, device=dev) for _ in range(2)]
    new, free = torch.full((3,), 20, dtype=torch.int32, device=dev), torch.arange(100, 120, dtype=torch.int32, device=dev)

    def both(i):
        q, k, v = qkv[i]
        a, b = S.apply_norm_rotary(q, k, pos, rot)
        return (a, b, S.compute_packed_attention(a, b, v, starts, score_cap=20.0),
                S.compute_paged_attention(a[:3], kv[0], kv[1], table, lens[i], 4000),
                *S.build_page_step(ctx[i], new, tables[i], free, 16, 64), tables[i].clone())
    want = [both(0), both(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(both(i))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(outs, want[i]))


@pytest.mark.parametrize("kw", [dict(score_cap=1e-20, scale=1e30), dict(score_cap=1e-30), dict(score_cap=9e29)])
def test_caps_at_the_ends_of_their_range(dev, kw):
    """Queries of 0 score 0 under any cap: the mean of the values, each weight exact, half a step of rounding."""
    q, k, v = (torch.randn(64, 2, 64, generator=_gen(44), device=dev).half() for _ in range(3))
    q.zero_()
    kv = torch.stack([k, v]).view(2, 4, 16, 2, 64)
    packed = S.compute_packed_attention(q, k, v, _starts([64], dev), causal=False, **kw)
    paged = S.compute_paged_attention(q[:1], kv[0], kv[1], torch.arange(4, dtype=torch.int32, device=dev)[None],
                                      torch.tensor([64], device=dev), 64, **kw)
    ref = v.double().mean(0)
    # sums of 64 products of at most max|v| in fp32, then one rounding
    tol = 2.0 ** -11 * ref.abs() + 64 * 2.0 ** -24 * v.double().abs().amax() + 2.0 ** -25
    for out in (*packed, paged[0]):
        _close(out, ref, tol, str(kw))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kw", [dict(score_cap=50.0), dict(score_cap=2.0), dict(slopes=True),
                                dict(score_cap=20.0, slopes=True), dict(window=33, score_cap=50.0)])
def test_packed_unseen_places_under_caps_and_biases(dev, kw, D):
    """NaN, infinities and numbers whose products overflow above a row and in other documents leave its bits."""
    kw, lens, at = dict(kw), [70, 300, 90], 70 + 171
    if kw.pop("slopes", False):
        kw["alibi_slopes"] = torch.tensor([0.5, 0.01], device=dev)
    q, k, v = _qkv(dev, 460, 2, 1, D, torch.bfloat16, 46)
    clean = S.compute_packed_attention(q, k, v, _starts(lens, dev), **kw)
    for bad in (float("nan"), INF, -INF, 3e38):
        for which in "kv":
            x = {"k": k.clone(), "v": v.clone()}
            x[which][at:370] = bad
            got = S.compute_packed_attention(q, x["k"], x["v"], _starts(lens, dev), **kw)
            assert torch.equal(got[:at], clean[:at]) and torch.equal(got[370:], clean[370:]), (bad, which)


@pytest.mark.parametrize("n", [65535, 1000003])
def test_very_many_documents_of_one_token(dev, n):
    """A token that sees itself alone has its value, bit for bit."""
    q, k, v = _qkv(dev, n, 2, 1, 8, torch.float16, 48)
    out = S.compute_packed_attention(q, k, v, torch.arange(n + 1, device=dev), score_cap=30.0)
    assert torch.equal(out, v.expand(-1, 2, -1))


@pytest.mark.parametrize("longest", [16, 400])
def test_the_most_sequences(dev, longest):
    """65535 sequences, most of them empty or of one token; the rest see equal keys, and so the mean of their values."""
    n, d = 65535, 8
    lens = torch.ones(n, dtype=torch.int32, device=dev)
    lens[::7] = 0
    lens[5::9973] = longest
    kv = torch.zeros(2, 40, 16, 1, d, dtype=torch.float16, device=dev)
    kv[1] = torch.randn(40, 16, 1, d, generator=_gen(49), device=dev).half()
    table = torch.randint(0, 40, (n, (longest + 15) // 16), generator=_gen(50), device=dev)
    q = torch.randn(n, 2, d, generator=_gen(51), device=dev).half()
    out = S.compute_paged_attention(q, kv[0], kv[1], table, lens, longest)
    first = kv[1][table[:, 0], 0, 0]
    assert bool((out[lens == 0] == 0).all())
    one = lens == 1
    assert torch.equal(out[one], first[one][:, None].expand(-1, 2, -1))
    for b in torch.nonzero(lens == longest).flatten().tolist():
        seen = kv[1][table[b]].reshape(-1, d)[:longest].double()
        ref = seen.mean(0)
        # weights of 1; a sum of `longest` values in fp32, one rounding
        tol = 2.0 ** -11 * ref.abs() + longest * 2.0 ** -24 * seen.abs().amax() + 2.0 ** -25
        _close(out[b], ref.expand(2, -1), tol.expand(2, -1), f"sequence {b}")


def test_the_largest_page_step(dev):
    """8000 requests with long contexts and the longest blocks: slots beyond 32 bits."""
    n, bs = 8000, 65536
    ctx = torch.full((n,), 70000, dtype=torch.int64, device=dev)
    new = torch.full((n,), 3, dtype=torch.int32, device=dev)
    table = torch.full((n, 2), 2 ** 31 - 1, dtype=torch.int32, device=dev)
    step = S.build_page_step(ctx, new, table, torch.empty(0, dtype=torch.int32, device=dev), bs, 3 * n)
    want = (2 ** 31 - 1) * bs + 70000 - bs
    assert step.slot_mapping.view(n, 3).tolist() == [[want, want + 1, want + 2]] * n
    assert step.status.tolist() == [0, 0] and int(step.query_start_loc[-1]) == 3 * n


@pytest.mark.parametrize("kw", [dict(), dict(causal=False), dict(prefix=[40, 200, 1]), dict(window=50),
                                dict(prefix=[3, 150, 90], window=20, cap=30.0)])
def test_packed_biases_in_every_mask(dev, kw):
    """Keys behind a row, which prefixes and full masks show it, are biased by their distance too."""
    _check_packed(dev, [100, 260, 91], 4, 2, 128, torch.bfloat16, slopes=torch.tensor([0.6, 0.1, -0.05, 0.0], device=dev),
                  **kw)


@pytest.mark.parametrize("slope", [1e4, 1e24, 1e30, 1e37])
def test_packed_steep_biases(dev, slope):
    """A bias that leaves a row nothing but its own key: its value, bit for bit."""
    q, k, v = _qkv(dev, 300, 2, 1, 64, torch.bfloat16, 52)
    out = S.compute_packed_attention(q, k, v, _starts([300], dev), alibi_slopes=torch.full((2,), slope, device=dev))
    assert torch.equal(out, v.expand(-1, 2, -1))
