"""The router over every count of workgroups: one, up to 512 that sum the counts of
the others themselves, and more, whose counts a launch of its own sums; with logits of
each type, experts that are masked or NaN or infinite among them. The tolerances are
those derived in test_experts_gpu.py."""
import math

import pytest

from test_experts_gpu import FLOOR, HALF_UNIT, _assert_within, _dtype, _gen, _normal, _route, _torch

import mini_triton_nvgpu_v1_amd as tb

pytestmark = pytest.mark.gpu


def _reference(x, top_k, renormalize):
    """ids, weights (NaN where a token has a NaN or +inf), slots, rows, offsets and the
    softmax in 64 bits."""
    torch = _torch()
    tokens, experts = x.shape
    d = x.double().nan_to_num(-math.inf, math.inf, -math.inf)
    top, ids = torch.sort(d, dim=1, descending=True, stable=True)
    top, ids = top[:, :top_k], ids[:, :top_k]
    ok = top > -math.inf
    odd = (x.isnan() | (x == math.inf)).any(1)
    pool = d
    if renormalize:
        pool = torch.full_like(d, -math.inf).scatter(1, ids, top)
    m = pool.amax(1, keepdim=True)
    z = torch.where(pool > -math.inf, torch.exp(pool - torch.where(m > -math.inf, m, 0.0)), 0.0)
    p = z / z.sum(1, keepdim=True).clamp_min(1e-300)
    p[odd] = math.nan
    w = torch.where(ok, p.gather(1, ids), 0.0)
    # pairs by expert, then by token
    token = torch.arange(tokens, device=x.device)[:, None].expand_as(ids)
    key = torch.where(ok, ids * tokens + token, experts * tokens).flatten()
    order = torch.sort(key, stable=True).indices
    used = int(ok.sum())
    slots = torch.full((tokens * top_k,), -1, dtype=torch.int32, device=x.device)
    slots[order[:used]] = torch.arange(used, dtype=torch.int32, device=x.device)
    rows = torch.full_like(slots, -1)
    rows[:used] = (order[:used] // top_k).to(torch.int32)
    counts = torch.bincount(ids[ok], minlength=experts)
    offsets = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).to(torch.int32)
    ids = torch.where(ok, ids, -1).to(torch.int32)
    return ids, w, slots.view(tokens, top_k), rows, offsets, p, odd


def _check(tokens, experts, top_k, dtype, renormalize, masked):
    torch = _torch()
    g = _gen(tokens * 1000 + experts)
    x = _normal(g, tokens, experts, scale=2.0).to(_dtype(dtype))
    if masked:
        hide = torch.rand((tokens, experts), generator=g, device="cuda") < masked
        hide[::5] = True  # tokens that nothing is left of
        x = x.masked_fill(hide, -math.inf)
    if tokens > 3:
        x[tokens // 2, experts // 2] = math.nan
        x[tokens - 1, 0] = math.inf
        x[tokens - 2] = torch.finfo(x.dtype).min  # the type's lowest value is no mask
    got = _route(x, top_k, renormalize)
    ids, w, slots, rows, offsets, p, odd = _reference(x, top_k, renormalize)
    assert torch.equal(got["offsets"], offsets)
    assert torch.equal(got["ids"], ids)
    assert torch.equal(got["slots"], slots)
    assert torch.equal(got["rows"], rows)
    none = ids < 0
    assert (got["weights"][none] == 0).all()
    assert got["weights"][odd][~none[odd]].isnan().all()
    w = torch.where(none, 0.0, w)
    _assert_within(got["weights"][~odd], w[~odd], (experts + 32) * 2.0 ** -24 * w[~odd] + 1e-30,
                   "weights")
    dw = _normal(g, tokens, top_k)
    dx = torch.full_like(x, math.nan)
    tb.route_backward(dw, x, got["ids"], dx, renormalize=renormalize)
    full = torch.zeros((tokens, experts + 1), dtype=torch.float64, device="cuda")
    full.scatter_(1, torch.where(none, experts, ids.long()), dw.double())
    full = full[:, :experts]
    assert dx[odd].gather(1, ids[odd].clamp_min(0).long())[~none[odd]].isnan().all()
    p, full, dx = p[~odd], full[~odd], dx[~odd]
    dot = (full * p).sum(1, keepdim=True)
    want = p * (full - dot)
    size = p * (full.abs() + (full * p).abs().sum(1, keepdim=True))
    bound = ((2 * experts + 64) * 2.0 ** -24 * size + HALF_UNIT[dtype] * want.abs()
             + FLOOR[dtype] + 1e-30)
    _assert_within(dx, want, bound, "dlogits")


@pytest.mark.parametrize("tokens, experts, top_k", [
    (1, 1, 1), (1, 8, 8), (13, 64, 6), (63, 65, 4), (65, 129, 1), (256, 16, 2), (257, 16, 2),
    (300, 512, 32), (40, 300, 17), (1000, 60, 5), (4097, 128, 8)])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("masked", [0.0, 0.7])
def test_route_f16(device, tokens, experts, top_k, renormalize, masked):
    _check(tokens, experts, top_k, "f16", renormalize, masked)


@pytest.mark.parametrize("tokens, experts, top_k", [
    (257, 128, 8), (5000, 300, 20), (32704, 60, 4), (32768, 60, 4), (32769, 60, 4),
    (33000, 1, 1), (40001, 65, 3), (70001, 512, 8)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("renormalize, masked", [(True, 0.0), (False, 0.6)])
def test_route_many_tokens(device, tokens, experts, top_k, dtype, renormalize, masked):
    """512 blocks of 64 tokens are the last whose counts the placing step sums."""
    _check(tokens, experts, top_k, dtype, renormalize, masked)
