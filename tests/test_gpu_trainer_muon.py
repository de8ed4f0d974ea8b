"""Muon inside the joint training step: the hidden matrices against float64
Newton-Schulz of the step's own gradients, everything else against Adam.

Tolerance: 4e-4 of the update's norm, the bound of the Newton-Schulz tests for
spread singular values, and the parameter's own roundings (two of 2^-24 a
step); Adam's elements as in the optimiser's own test (1e-6)."""
import numpy as np
import pytest

from yumelayers_b200 import ops, synth
from yumelayers_b200._lib import YumeError

pytestmark = pytest.mark.gpu
FIRST_LAST = {0: ("enc.conv_in.weight", "dec.conv_out.weight"),
              1: ("conv_in.weight", "conv_out.weight")}


def r4(v):
    return (v + 3) & ~3


def ns64(x, steps=5):
    flip = x.shape[0] > x.shape[1]
    x = (x.T if flip else x).astype(np.float64)
    x = x / (np.linalg.norm(x) + 1e-7)
    for _ in range(steps):
        g = x @ x.T
        x = 3.4445 * x - 4.7750 * (g @ x) + 2.0315 * (g @ (g @ x))
    return x.T if flip else x


def trainer(seed=1, **kw):
    from yumelayers_b200.trainer import Trainer, default_config
    return Trainer(default_config(batch=1, height=32, width=48, seed=seed, **kw))


def batches(n):
    clips = [synth.make_clip(21, h=32, w=48, width_padded=48)]
    return [synth.sample_batch(clips, 1, seed=s) for s in range(n)]


def hidden(table, which):
    """(offset, stored rows, stored columns, scale) of the matrices Muon updates."""
    out = []
    for e in table:
        if not e.name.endswith(".weight") or e.name in FIRST_LAST[which]:
            continue
        oc, ic, k1, k2 = e.shape
        rows, cols, logical = (oc, ic, ic) if k1 == 0 else (r4(oc), k1 * k2 * r4(ic), ic * k1 * k2)
        out.append((e.offset, rows, cols, ops.muon_scale(oc, logical)))
    return out


@pytest.mark.parametrize("clip", [0.0, 0.05])
def test_step_matches_definition(clip):
    tr = trainer(clip_max_norm=clip)
    bs = batches(2)
    tr.set_muon(lr_vae=0.01, lr_motion=0.02, momentum=0.9, nesterov=True, weight_decay=0.05)
    tr.step_host(*bs[0])  # momenta and moments that are not zero
    before = {w: [tr.download(w, k).astype(np.float64) for k in range(4)] for w in (0, 1)}
    tr.step_host(*bs[1])
    for w, lr in ((0, 0.01), (1, 0.02)):
        p0, _, m0, v0 = before[w]
        p, g, m, v = (tr.download(w, k).astype(np.float64) for k in range(4))
        if clip:
            norm = np.linalg.norm(g)
            assert norm > clip
            g = g * (clip / norm)
        rest = np.ones(p.size, bool)
        mats = hidden(tr.param_table(w), w)
        assert len(mats) > 20
        for o, r, c, scale in mats:
            at = slice(o, o + r * c)
            rest[at] = False
            mm = 0.9 * m0[at] + g[at]
            assert np.linalg.norm(m[at] - mm) < 1e-6 * np.linalg.norm(mm)
            assert np.array_equal(v[at], v0[at])
            u = (g[at] + 0.9 * mm).reshape(r, c)
            step = lr * scale * ns64(u).reshape(-1)
            want = p0[at] * (1 - lr * 0.05) - step
            assert np.linalg.norm(p[at] - want) < 4e-4 * np.linalg.norm(step) + 1.5e-7 * np.linalg.norm(want)
        mm = 0.9 * m0[rest] + 0.1 * g[rest]
        vv = 0.999 * v0[rest] + 0.001 * g[rest] ** 2
        want = p0[rest] - 2e-4 * (mm / (1 - 0.9 ** 2)) / (np.sqrt(vv / (1 - 0.999 ** 2)) + 1e-8)
        assert np.abs(p[rest] - want).max() < 1e-6
    tr.close()


def test_muon_resumes_bit_identically_and_adam_comes_back(tmp_path):
    from yumelayers_b200 import checkpoint as ck
    bs = batches(4)
    a = trainer(seed=3)
    a.set_muon(lr_vae=0.005, lr_motion=0.01)
    for b in bs[:2]:
        a.step_host(*b)
    ck.save_trainer(a, tmp_path / "v.safetensors", tmp_path / "m.safetensors", epoch=1)
    c = trainer(seed=4)
    ck.load_trainer(c, tmp_path / "v.safetensors", tmp_path / "m.safetensors")
    assert c.muon == a.muon and c.step == 2
    for tr in (a, c):
        tr.step_host(*bs[2])
        tr.unset_muon()
        tr.step_host(*bs[3])
    for w in (0, 1):
        for kind in (0, 2, 3):
            np.testing.assert_array_equal(a.download(w, kind), c.download(w, kind))
    a.close()
    c.close()


def test_unset_before_a_step_leaves_adam_as_it_was():
    bs = batches(2)
    a, b = trainer(seed=5), trainer(seed=5)
    b.set_muon()
    b.unset_muon()
    for x in bs:
        a.step_host(*x)
        b.step_host(*x)
    for w in (0, 1):
        np.testing.assert_array_equal(a.download(w), b.download(w))
    a.close()
    b.close()


def test_refused_settings():
    tr = trainer(seed=6)
    for bad in (dict(momentum=1.0), dict(momentum=-0.1), dict(steps=0), dict(steps=33),
                dict(lr_vae=float("nan")), dict(weight_decay=-1.0),
                dict(lr_motion=float("inf"))):
        with pytest.raises(YumeError):
            tr.set_muon(**bad)
        assert tr.muon is None
    tr.close()
