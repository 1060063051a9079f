"""Gradients that are strided views: whether two of them share memory is decided by their elements, not by where they start, and nothing is scaled before a refusal."""
import itertools

import pytest
import torch

from cagc.op import clip_grad_norm_, get_total_norm
from cagc.op.grad_clip import _share_memory

gpu = pytest.mark.gpu


def params_with(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(g.shape, dtype=g.dtype, device=g.device))
        p.grad = g
        out.append(p)
    return out


def views(base):
    """many views of one buffer of 240 elements"""
    v = [base[a:a + n] for a, n in ((0, 240), (0, 10), (5, 10), (10, 1), (239, 1))]
    m = base.view(12, 20)
    v += [m[:, 0:3], m[:, 2:5], m[:, 3:5], m[:, ::2], m[:, 1::2], m[::2], m[1::2], m[::3, 1:4], m[:5, 7:9], m[5:, 7:9], m[3:4, 4:9], m.t()[4:6], m[:, 19:], m[1:, :1]]
    c = base.view(3, 4, 4, 5)
    v += [c[:, 1], c[:, 2:], c[:, :, 1:3, 2], c[:, ::2, ::2, ::2], c[:, 1::2, 1::2], c.permute(0, 2, 3, 1), c[..., 4], c[1, 2, 3]]
    v += [base.as_strided(*s) for s in (((6, 4), (7, 3), 2), ((5, 3), (9, 2), 100), ((4, 5), (6, 1), 3), ((3, 3), (2, 2), 50), ((4,), (0,), 8), ((2, 3), (0, 5), 40), ((8, 5), (13, 2), 1))]
    return v


def elements(t, base):
    return set(torch.arange(base.numel()).as_strided(t.size(), t.stride(), t.storage_offset()).reshape(-1).tolist())


def test_by_elements():
    base = torch.zeros(240)
    vs = views(base)
    for a, b in itertools.combinations(vs, 2):
        assert _share_memory([a, b]) == bool(elements(a, base) & elements(b, base)), (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
    assert _share_memory([vs[0], vs[0]]) and not _share_memory([vs[0]]) and not _share_memory([base[:0], base, base[3:3]])


def test_of_different_types():
    raw = torch.zeros(960, dtype=torch.uint8)
    f, h = raw.view(torch.float32).view(12, 20), raw.view(torch.float16).view(24, 20)
    assert _share_memory([f[:, :3], h[0:2, 4:6]]) and not _share_memory([f[:, :3], h[::2, 6:9]]) and not _share_memory([f[1::2, 2:4], h[::4]])


def test_many_columns_of_one_buffer():
    base = torch.zeros(100, 64 * 7)
    cols = list(base.split(7, 1))
    assert not _share_memory(cols) and _share_memory(cols + [base[99:, 300:302]])


@gpu
def test_overlapping_views_are_refused_before_anything_changes():
    base = torch.randn(40, 30, device="cuda")
    keep = base.clone()
    own = torch.randn(50, device="cuda")
    own0 = own.clone()
    row = torch.randn(1, 8, device="cuda")
    for bad in ([own, base[:, 0:3], base[:, 2:5]], [own, base[3], base[:, 2:5]], [own, base, base[:, ::2]], [own, base.view(-1)[7:900], base[::2, 4:6]]):
        with pytest.raises(RuntimeError, match="share memory"):
            clip_grad_norm_(params_with(bad), 0.1)
        with pytest.raises(RuntimeError, match="share memory"):
            get_total_norm(bad)
        assert torch.equal(base, keep) and torch.equal(own, own0)
    with pytest.raises(RuntimeError, match="share memory"):      # an expanded gradient's own elements share memory
        clip_grad_norm_(params_with([own, row.expand(5, 8)]), 0.1)
    assert torch.equal(own, own0)
    want = float((own.double().square().sum() + 5 * row.double().square().sum()).sqrt())
    assert abs(float(get_total_norm([own, row.expand(5, 8)])) - want) <= 2.0 ** -23 * want


@gpu
def test_views_apart_are_clipped():
    base = torch.randn(40, 30, device="cuda")
    before = base.double().cpu()
    grads = [base[:, 0:3], base[:, 3:5], base[::2, 5::2], base[1::2, 6:9]]
    touched = torch.zeros(40, 30, dtype=torch.bool)
    touched[:, :5] = True
    touched[::2, 5::2] = True
    touched[1::2, 6:9] = True
    total = float(before[touched].square().sum().sqrt())
    norm = clip_grad_norm_(params_with(grads), 0.25 * total)
    assert abs(float(norm) - total) <= 2.0 ** -23 * total
    want = torch.where(touched, before * (0.25 * total / (total + 1e-6)), before)
    assert bool(((base.double().cpu() - want).abs() <= want.abs() * 4 * 2.0 ** -24).all())
