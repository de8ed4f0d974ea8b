"""The driver's warm-up with a trainer that has Muon set."""

import numpy as np

from test_driver import FakeTrainer, _batch
from yumelayers_b200 import driver as dv


def test_warmup_ramps_muon_rates_too():
    class WithMuon(FakeTrainer):
        def __init__(self, losses):
            super().__init__(losses)
            self.muon = dict(lr_vae=0.02, lr_motion=0.04, momentum=0.9)
            self.muon_rates = []

        def set_muon(self, **kw):
            self.muon = kw

        def step_host(self, frames, t):
            self.muon_rates.append((self.muon["lr_vae"], self.muon["lr_motion"]))
            assert self.muon["momentum"] == 0.9
            return super().step_host(frames, t)

    tr = WithMuon([[1.0, 0.5]] * 3)
    dv.run_training(tr, _batch, epochs=1, epoch_steps=3, warmup_steps=2)
    np.testing.assert_allclose(tr.muon_rates, [(0.01, 0.02), (0.02, 0.04), (0.02, 0.04)])
    assert tr.muon["lr_vae"] == 0.02


def test_checkpoints_during_warmup_keep_the_full_muon_rates():
    class WithMuon(FakeTrainer):
        muon = dict(lr_vae=0.02, lr_motion=0.04)

        def set_muon(self, **kw):
            self.muon = kw

    tr, saved = WithMuon([[1.0, 0.5]] * 4), []
    dv.run_training(tr, _batch, epochs=2, epoch_steps=2, warmup_steps=8, save_every=1,
                    save=lambda *at: saved.append((at, dict(tr.muon))))
    assert [at for at, _ in saved] == [(0, 1), (1, 0), (1, 1), (2, 0)]
    assert all(m == dict(lr_vae=0.02, lr_motion=0.04) for _, m in saved)
