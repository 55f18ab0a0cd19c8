"""Blocks with a norm on a sublayer's output, in front of a feed-forward whose first matrix is in 8 bits: the one kernel that ends the mixer's part (its norm, the stream's sum) also
leaves the feed-forward's rows in 8 bits, rounded once, from the stream or the next norm's rows as float32 has them.

Bounds: the stream and the rows before 8 bits 64 steps of 2^-24 of what is added (a sum of 192 squares, a root, a division), the rows half a step of e4m3 beside that."""
import importlib

import numpy as np
import pytest
import torch

import plain_blocks8 as p8

pytestmark = pytest.mark.gpu
K = importlib.import_module("daisi-llogos_amd.ops.kernels")
base = importlib.import_module("daisi-llogos_amd.parts.base")
block = importlib.import_module("daisi-llogos_amd.parts.block")
norms = importlib.import_module("daisi-llogos_amd.parts.norm")
BF16 = torch.bfloat16
H = 192
RT = base.Runtime(torch.device("cuda:0"), BF16, eight_bit=True)


class Gives(base.Mixer):
    """A mixer that gives what it is told to."""

    def __init__(self, out):
        self.out = out

    def forward(self, ctx, h, cache):
        return self.out

    def caches_of(self, caches):
        return None

    def cache_parts(self):
        return []


class Takes(base.FeedForward):
    """A feed-forward that keeps its rows and gives what it is told to."""

    def __init__(self, out, eight):
        self.out, self.takes_block_rows, self.rows = out, eight, None

    def forward(self, ctx, h):
        self.rows = h
        return self.out


def norm(name, seed, eps, kind="rms"):
    g = torch.Generator().manual_seed(seed)
    n = norms.RMSNorm(name, H, eps) if kind == "rms" else norms.LayerNorm(name, H, eps)
    w = 1.0 + 0.3 * torch.randn(H, generator=g)
    n.bind(lambda _: w, RT)
    return n


def arrangement(kind, a, d, eight, eps=(1e-5, 1e-6), of="rms"):
    parts = [norm(str(i), i, eps[i % 2], of) for i in range(4)]
    if kind == "output":
        b = block.OutputNormBlock(parts[0], Gives(a), parts[1], Takes(d, eight))
    else:
        b = block.SandwichBlock(parts[0], Gives(a), parts[1], parts[2], Takes(d, eight), parts[3])
    b.rt = RT
    return b


CTX = base.StepContext(RT, 5, 1, *[None] * 4, [0, 5], [0], [0], False, 5)


@pytest.mark.parametrize("T,what", [(5, BF16), (5, torch.float32), (3, "parts"), (70, "parts"), (300, BF16), (1, BF16)])
@pytest.mark.parametrize("kind", ["output", "sandwich"])
def test_rows_behind_a_norm_on_the_output(kind, T, what):
    g = torch.Generator(device="cuda").manual_seed(T)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x0, d = r(T, H) * 3, r(T, H).to(BF16)
    a = r(3, T, H) if what == "parts" else r(T, H).to(what)
    x, b = x0.clone(), arrangement(kind, a, d, True)
    x, pending = b.forward(CTX, x, None, [])
    rows = b.ffn.rows
    assert isinstance(rows, K.BlockRows) and rows.shape == (T, H)
    # the plain form in 64 bits
    n = lambda t: t.double().cpu().numpy()  # noqa: E731
    out = n(a).sum(axis=0) if what == "parts" else n(a)
    post = b.mixer_norm if kind == "output" else b.post_mixer_norm
    stream = n(x0) + p8.rmsnorm(out, n(post.weight), post.eps)
    want = stream if kind == "output" else p8.rmsnorm(stream, n(b.ffn_norm.weight), b.ffn_norm.eps)
    size = np.abs(n(x0)) + np.abs(stream - n(x0)) + 1
    off = 64 * 2.0 ** -24 * (size if kind == "output" else size * np.abs(want).max() / np.abs(stream).max() * 4)
    step = np.repeat(n(rows.powers.float()), 128, axis=1)[:, :H]
    assert (np.abs(n(rows.values()) - want) <= np.maximum(2.0 ** -4 * (np.abs(want) + off), 2.0 ** -10 * step) + off).all()
    last = b.ffn_norm if kind == "output" else b.post_ffn_norm
    stream = stream + p8.rmsnorm(n(d), n(last.weight), last.eps)
    assert (np.abs(n(x) - stream) <= 64 * 2.0 ** -24 * (size + np.abs(stream))).all()
    # and what the stream and the rest come to where the feed-forward takes them in bfloat16
    y, c = x0.clone(), arrangement(kind, a, d, False)
    y, other = c.forward(CTX, y, None, [])
    assert c.ffn.rows.dtype == BF16 and (np.abs(n(y) - n(x)) <= 128 * 2.0 ** -24 * (size + np.abs(stream))).all()
    assert type(other) is type(pending)


@pytest.mark.parametrize("kind", ["output", "sandwich"])
def test_other_norms_keep_their_own_kernels(kind):
    """A layer norm has no such kernel: the feed-forward gets rows in bfloat16, and brings them to 8 bits itself."""
    g = torch.Generator(device="cuda").manual_seed(1)
    a, d, x = (torch.randn(4, H, generator=g, device="cuda") for _ in range(3))
    b = arrangement(kind, a.to(BF16), d.to(BF16), True, of="layer")
    b.forward(CTX, x, None, [])
    assert isinstance(b.ffn.rows, torch.Tensor) and b.ffn.rows.dtype == BF16
