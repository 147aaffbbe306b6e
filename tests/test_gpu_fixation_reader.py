"""GPU: the token operators together, as FixationReader runs them behind the sensor and the patch embedding."""
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from conftest import synth_images

pytestmark = pytest.mark.gpu


def _reader(dim=96, heads=3, kv_heads=None, queries=2, depth=2):
    from fovi_b200.knn import KNNPartitioningPatchEmbedding
    from fovi_b200.sensing import RetinalTransform
    from fovi_b200.tokens import FixationReader
    torch.manual_seed(3)
    retina = RetinalTransform(64, start_res=64, fov=16, cmf_a=2.78, sampler="grid_bilinear")
    embedding = KNNPartitioningPatchEmbedding(3, dim, in_res=retina.resolution, fov=16, cmf_a=2.78, in_cart_res=64, cart_patch_size=8, ref_frame_side_length=16, bias=True,
                                              auto_match_cart_resources=0)
    with torch.no_grad():
        embedding.weight.normal_(0, (1 / embedding.weight.shape[1]) ** 0.5)
        embedding.bias.normal_(0, 0.1)
    return FixationReader(retina, embedding, dim, heads, 10, queries=queries, depth=depth, kv_heads=kv_heads).cuda()


def _plain_read(m, states, places, counts=None):
    """m.read in 64 bits, with torch's own layer norm and softmax."""
    per = len(m.embedding.out_coords)
    states, places = states.double(), places.double()
    norm = lambda n, x: F.layer_norm(x, x.shape[-1:], n.weight.double(), n.bias.double(), n.eps)  # noqa: E731
    lin = lambda l, x: F.linear(x, l.weight.double(), l.bias.double())  # noqa: E731
    P = m.rotary.frequencies.numel()
    axis = [a for a, n in enumerate(m.rotary.pairs_per_axis) for _ in range(n)]
    t = places[..., axis] * m.rotary.frequencies.double()
    t = t[:, :, None]
    x = m.queries.double().expand(states.shape[0], -1, -1)
    for n, b in zip(m.norms, m.blocks):
        q = lin(b.query, norm(n, x)).unflatten(-1, (b.heads, -1))
        k, v = (lin(l, states).unflatten(-1, (b.kv_heads, -1)) for l in (b.key, b.value))
        u, w, rest = k[..., :P], k[..., P:2 * P], k[..., 2 * P:]
        k = torch.cat([u * t.cos() - w * t.sin(), w * t.cos() + u * t.sin(), rest], -1)
        k, v = (z.repeat_interleave(b.heads // b.kv_heads, 2) for z in (k, v))
        s = torch.einsum("bqhd,bkhd->bhqk", q, k) / math.sqrt(b.head_dim)
        if counts is not None:
            s = s.masked_fill((torch.arange(s.shape[-1], device=s.device) >= counts[:, None] * per)[:, None, None], float("-inf"))
        x = x + lin(b.out, torch.einsum("bhqk,bkhd->bqhd", s.softmax(-1), v).flatten(2))
    return lin(m.classifier, norm(m.norm, x).mean(1))


def _images():
    images = torch.from_numpy(synth_images(4, (3, 3, 64, 64))).cuda()
    fix = torch.from_numpy(np.random.RandomState(5).uniform(0.25, 0.75, (3, 4, 2)).astype(np.float32)).cuda()
    return images, fix


@pytest.mark.autograd
@pytest.mark.parametrize("kv_heads", [None, 1])
def test_reading_and_its_gradients(kv_heads):
    """Scores and all gradients against the same model in 64 bits.  The projections are float32 library products: 1e-5 of the result's size."""
    m = _reader(kv_heads=kv_heads)
    images, fix = _images()
    with torch.no_grad():
        states, places = m.states(images, fix)
    assert states.shape == (3, 4 * len(m.embedding.out_coords), 96) and places.shape == states.shape[:2] + (3,)
    counts = torch.tensor([4, 1, 3], device="cuda")
    params = [m.queries] + [p for mod in (m.norms, m.blocks, m.norm, m.classifier) for p in mod.parameters()]
    g = torch.randn(3, 10, device="cuda")
    leaf = states.requires_grad_(True)
    got = m.read(leaf, places, counts * len(m.embedding.out_coords))
    grads = torch.autograd.grad(got, [leaf] + params, g)
    want = _plain_read(m, leaf, places, counts)
    wants = torch.autograd.grad(want, [leaf] + params, g.double())
    for a, b in zip((got,) + grads, (want,) + wants):
        # a query's gradient that vanishes by symmetry (the key's bias) is compared on the scale of the others
        scale = max(b.double().norm().item(), 1e-3 * max(w.double().norm().item() for w in wants))
        assert (a.double() - b.double()).norm().item() <= 1e-5 * scale


@pytest.mark.autograd
def test_training_from_images_and_counts():
    """Every parameter gets a gradient; an image with one fixation that counts is the image with that fixation alone."""
    m = _reader()
    images, fix = _images()
    m(images, fix).square().sum().backward()
    for name, p in m.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
        assert p.grad.abs().max() > 0 or name.endswith("key.bias"), name
    with torch.no_grad():
        few = m(images, fix, fixation_counts=torch.ones(3, dtype=torch.int64, device="cuda"))
        alone = m(images, fix[:, :1])
    assert (few - alone).norm() <= 1e-5 * alone.norm()


def test_under_autocast():
    """bf16 projections and attention: within 2e-2 of the float32 scores."""
    m = _reader(dim=128, heads=2)
    images, fix = _images()
    want = m(images, fix)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = m(images, fix)
    assert (got.float() - want).norm() <= 2e-2 * want.norm()


def test_places():
    m = _reader()
    images, fix = _images()
    _, places = m.states(images, fix, fixation_size=32)
    n = len(m.embedding.out_coords)
    xy = m.embedding.out_coords.cartesian.cuda()
    p = places.view(3, 4, n, 3)
    assert torch.equal(p[..., 0], torch.arange(4.0, device="cuda").view(1, 4, 1).expand(3, 4, n))
    want = 2 * fix[:, :, None] - 1 + torch.stack([-xy[:, 1], xy[:, 0]], 1) * 0.5
    assert torch.allclose(p[..., 1:], want, atol=1e-6)
