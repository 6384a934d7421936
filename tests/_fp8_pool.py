"""Shared setup of the 8-bit pool's tests: a pool on the GPU and the same pool for the oracle."""
from __future__ import annotations

import numpy as np
import torch

FP8 = torch.float8_e4m3fn


class Fp8Pool:
    """Random full blocks, shuffled tables; .args() are the entry points' pool arguments."""

    def __init__(self, lens, hkv, d, bs, seed, device, slack=2, spread=1.0, shared=None):
        rng = np.random.default_rng(seed)
        self.lens, self.hkv, self.d, self.bs = list(lens), hkv, d, bs
        need = [max(1, -(-n // bs)) for n in lens]
        self.blocks = sum(need) * slack + 3
        ids = rng.permutation(self.blocks)
        self.tables = np.zeros((len(lens), max(need, default=1)), dtype=np.int32)
        at = 0
        for i, n in enumerate(need):
            self.tables[i, :n] = ids[at:at + n]
            at += n
        if shared:  # every sequence's first blocks are the first one's
            self.tables[:, :shared] = self.tables[0, :shared]
        gen = torch.Generator().manual_seed(seed)
        self.k, self.k_scale = self._half(gen, spread)
        self.v, self.v_scale = self._half(gen, spread)
        self.device = device
        self.dk, self.dv = self.k.to(device), self.v.to(device)
        self.dks, self.dvs = self.k_scale.to(device), self.v_scale.to(device)
        self.dt = torch.from_numpy(self.tables).to(device)
        self.dl = torch.tensor(self.lens, dtype=torch.int32, device=device)

    def _half(self, gen, spread):
        """Codes that use their whole range, and scales around the ones of unit-normal rows."""
        x = torch.randn(self.blocks, self.bs, self.hkv, self.d, generator=gen)
        x *= 448 / x.abs().amax(dim=(1, 3), keepdim=True)
        e = torch.randint(-9, -6, (self.blocks, self.hkv), generator=gen).float() * spread
        return x.to(FP8), torch.exp2(e.round().clamp(-15, 8))

    def args(self):
        return self.dk, self.dv, self.dks, self.dvs, self.dt, self.dl

    def oracle(self):
        """float64 copies of the pool as it was set up."""
        return {"k": self.k.double().numpy(), "v": self.v.double().numpy(),
                "k_scale": self.k_scale.double().numpy(),
                "v_scale": self.v_scale.double().numpy()}

    def state(self):
        """The GPU pool's present codes (as values) and scales."""
        return {"k": self.dk.cpu().double().numpy(), "v": self.dv.cpu().double().numpy(),
                "k_scale": self.dks.cpu().double().numpy(),
                "v_scale": self.dvs.cpu().double().numpy()}


def starts_of(new):
    return [0, *np.cumsum(new).tolist()]


def int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)
