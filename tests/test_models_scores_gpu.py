"""``generate_scores`` / ``divergence`` through the network on the GPU: the operators on its logits, in the volume's layout."""
import numpy as np
import pytest

from dosma_amd import MedicalVolume
from dosma_amd import _lib as L
from dosma_amd.models import IWOAIOAIUnet2DNormalized, OAIUnet2D, StanfordQDessUNet2D
from oracle import answers_oracle as ao
from oracle import unet_oracle as uo

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
# 5 categories: the sums have 5 terms; log p = d - ln s with |d| the distance to the best logit (tests/test_answers_gpu.py)
AFFINE = np.array([[0, 0, 1.5, -40.0], [0, -0.4, 0, 60.0], [-0.4, 0, 0, 70.0], [0, 0, 0, 1.0]])


def tol(z, T):
    return U * (60 + 8 * (z.max(-1) - z.min(-1)) / T)


@pytest.fixture(scope="module")
def weights():
    return uo.make_weights(seed=3)


def volume(S=5, seed=9, H=64, W=32):
    v = (np.random.default_rng(seed).standard_normal((H, W, S)) * 80 + 200).astype(np.float32)
    return MedicalVolume(v, AFFINE)


def logits_of(model, v):
    """(H W S, categories) of the volume's voxels in its own order, the background in front."""
    x = np.ascontiguousarray(np.transpose(v.volume, (2, 0, 1)))
    z, _ = model.seg_model.forward_host(x, whiten=model._WHITEN, eps=model._WHITEN_EPS)
    return ao.with_background(np.transpose(z, (1, 2, 0, 3)).astype(np.float64).reshape(-1, z.shape[-1]))


@pytest.mark.parametrize("S, T, top", [(1, 1.0, 1), (5, 1.5, 3), (37, 0.7, 5)])
def test_scores_are_those_of_the_logits(weights, S, T, top):
    m = IWOAIOAIUnet2DNormalized((64, 32, 1), weights, force_weights=True)
    v = volume(S)
    lab = np.random.default_rng(S).integers(0, 5, v.shape).astype(np.uint8)
    lab[3:5] = 255
    r = m.generate_scores(v, top=top, temperature=T, labels=MedicalVolume(lab, AFFINE))
    z = logits_of(m, v)
    want = ao.scores(z, T, lab.reshape(-1).astype(int), top, ignore=255)
    t = tol(z, T)
    for k in range(top):
        assert np.array_equal(r.top_labels[k].volume.reshape(-1), want["top_label"][:, k])
        assert np.all(np.abs(r.top_log_probs[k].volume.reshape(-1) - want["top_log_prob"][:, k]) <= t)
    assert np.all(np.abs(r.log_prob.volume.reshape(-1) - want["log_prob"]) <= t)
    assert np.all(np.abs(r.entropy.volume.reshape(-1) - want["entropy"]) <= 4 * t)
    # the best label is where the masks say there is tissue at all
    masks = m.generate_mask(v)
    any_tissue = np.any([p.volume for p in masks.values()], axis=0)
    assert np.array_equal(r.top_labels[0].volume > 0, any_tissue)


def test_divergence_between_precisions(weights):
    v = volume(4)
    m = IWOAIOAIUnet2DNormalized((64, 32, 1), weights, force_weights=True)
    exact = m.generate_scores(v, top=2)
    assert np.abs(m.divergence(v, exact).volume).max() < 100 * U  # its own answers, as float32
    z1 = logits_of(m, v)
    m.seg_model.set_precision("bf16")
    d = m.divergence(v, exact)
    z2 = logits_of(m, v)
    lab = np.stack([p.volume.reshape(-1) for p in exact.top_labels], -1).astype(int)
    lp = np.stack([p.volume.reshape(-1) for p in exact.top_log_probs], -1).astype(float)
    want = ao.distill(z2, lab, lp, 1.0, True)["loss"]
    # q log q and q_t log q_t: roundings of values up to the distances of the logits, q_t = 1 - sum q with 2 + 8 of them times |log|
    lim = 4 * tol(z2, 1.0) + 20 * U * (2 + np.abs(np.log(np.maximum(1 - np.exp(lp).sum(-1), 1e-8))) + (z2.max(-1) - z2.min(-1)))
    assert np.all(np.abs(d.volume.reshape(-1) - want) <= lim)
    assert not np.array_equal(z1, z2) and d.volume.max() > 0


def test_single_class_model_and_many_slices(weights):
    """One class: its sigmoid; more slices than one pass takes."""
    w = dict(weights)
    w["head_kernel"], w["head_bias"] = weights["head_kernel"][..., :1].copy(), weights["head_bias"][:1].copy()

    class Small(OAIUnet2D):
        gpu_batch = 16

    m = Small((64, 32, 1), w)
    v = volume(41)
    r = m.generate_scores(v, top=2)
    z = logits_of(m, v)
    p1 = 1.0 / (1.0 + np.exp(-z[:, 1]))
    got = np.where(r.top_labels[0].volume.reshape(-1) == 1, r.top_log_probs[0].volume.reshape(-1), r.top_log_probs[1].volume.reshape(-1))
    assert np.all(np.abs(got - np.log(p1)) <= tol(z, 1.0))
    assert m.seg_model.max_batch < 41


def test_dual_echo_input(weights):
    m = StanfordQDessUNet2D((64, 32, 1), weights)
    e = (np.random.default_rng(4).standard_normal((64, 32, 3, 2)) * 50 + 120).astype(np.float32)
    r = m.generate_scores(MedicalVolume(e, AFFINE))
    rss = np.sqrt(np.sum(e.astype(np.float64) ** 2, axis=-1)).astype(np.float32)
    r3 = m.generate_scores(MedicalVolume(rss, AFFINE))
    assert r.entropy.shape == (64, 32, 3)
    assert np.allclose(r.entropy.volume, r3.entropy.volume, rtol=0, atol=1e-3)  # (whitened from float64 and float32 volumes)


def test_engine_refusals(weights):
    m = IWOAIOAIUnet2DNormalized((64, 32, 1), weights, force_weights=True)
    eng, v = m.seg_model, volume(2).volume
    for call, says in (
            (lambda: eng.score_volume(v[:10]), "built for slices"),
            (lambda: eng.score_volume(v, labels=np.zeros(v.shape, np.int32)), "uint8"),
            (lambda: eng.score_volume(v, labels=np.zeros((64, 32, 3), np.uint8)), "uint8"),
            (lambda: eng.score_volume(v, top=6), "categories"),
            (lambda: eng.score_volume(v, top=1, temperature=0.0), "temperature"),
            (lambda: eng.score_volume(v, teacher=(np.zeros((6,) + v.shape, np.uint8), np.zeros((6,) + v.shape, np.float32))), "categories"),
            (lambda: eng.score_volume(v, teacher=(np.zeros(v.shape, np.uint8), np.zeros(v.shape, np.float32))), "teacher")):
        with pytest.raises(ValueError, match=says):
            call()
    empty = eng.score_volume(np.zeros((64, 32, 0), np.float32), top=1)
    assert empty["top_label"].shape == (1, 64, 32, 0)
    assert L.load().qmri_unet2d_score_volume(None, None) == L.QMRI_ERR_ARG


def test_a_volume_too_large_for_the_memory_leaves_the_model_usable(weights):
    """The allocation is refused (17 TB, nothing is read), and the next volume finds its buffers."""
    m = IWOAIOAIUnet2DNormalized((64, 32, 1), weights, force_weights=True)
    eng, v = m.seg_model, volume(3)
    first = m.generate_scores(v, top=2)
    mask = m.generate_mask(v)["fc"].volume
    import torch

    x = torch.zeros((1, 64, 32), device="cuda")
    for _ in range(2):
        with pytest.raises(L.QmriError):
            eng.forward_device(x.data_ptr(), 2 ** 31 - 1, None, None, whiten=True)
        again = m.generate_scores(v, top=2)
        assert np.array_equal(again.entropy.volume, first.entropy.volume)
        assert np.array_equal(again.top_labels[1].volume, first.top_labels[1].volume)
        assert np.array_equal(m.generate_mask(v)["fc"].volume, mask)
