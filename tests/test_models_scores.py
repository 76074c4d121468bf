"""``generate_scores`` / ``divergence`` of the segmentation models without a GPU (a stand-in engine that works on the host with the
64-bit definitions): orientations, label volumes, refusals."""
import numpy as np
import pytest

from dosma_amd import MedicalVolume
from dosma_amd.models import IWOAIOAIUnet2DNormalized, StanfordQDessUNet2D
from dosma_amd.models.oaiunet2d import AnswerMaps, OAIUnet2D
from oracle import answers_oracle as ao

H, W, S = 6, 5, 4
AFFINE = np.array([[0, 0, 1.5, -40.0], [0, -0.4, 0, 60.0], [-0.4, 0, 0, 70.0], [0, 0, 0, 1.0]])


class StandIn:
    """Logits a_c * v + b_c; ``score_volume`` as the engine's, from the oracle."""

    H, W = H, W
    a, b = np.array([1.0, -0.5, 0.25, 2.0]), np.array([0.1, 0.4, -0.3, -1.0])

    def rows(self, v):
        return ao.with_background(v.astype(np.float64).reshape(-1, 1) * self.a + self.b)

    def score_volume(self, v, *, whiten, eps, temperature=1.0, labels=None, entropy=False, top=0, teacher=None):
        assert v.shape[:2] == (H, W)
        z = self.rows(v)
        out = {}
        s = ao.scores(z, temperature, None if labels is None else labels.reshape(-1), top, ignore=255)
        if labels is not None:
            out["log_prob"] = s["log_prob"].reshape(v.shape).astype(np.float32)
        if entropy:
            out["entropy"] = s["entropy"].reshape(v.shape).astype(np.float32)
        if top:
            out["top_label"] = np.moveaxis(s["top_label"], -1, 0).reshape(top, *v.shape).astype(np.uint8)
            out["top_log_prob"] = np.moveaxis(s["top_log_prob"], -1, 0).reshape(top, *v.shape).astype(np.float32)
        if teacher is not None:
            k = teacher[0].shape[0]
            lab = np.moveaxis(teacher[0].reshape(k, -1), 0, -1).astype(np.int64)
            lab[lab == 255] = -1
            d = ao.distill(z, lab, np.moveaxis(teacher[1].reshape(k, -1), 0, -1), temperature, True)
            out["divergence"] = d["loss"].reshape(v.shape).astype(np.float32)
        return out

    def close(self):
        pass


class Model(IWOAIOAIUnet2DNormalized):
    def __init__(self):
        self.seg_model = StandIn()


def volume(seed=0):
    return MedicalVolume(np.random.default_rng(seed).standard_normal((H, W, S)).astype(np.float32), AFFINE)


def test_scores_in_the_volumes_orientation():
    m, v = Model(), volume()
    assert v.orientation == ("SI", "AP", "LR")
    r = m.generate_scores(v, top=3, temperature=1.5)
    assert isinstance(r, AnswerMaps) and len(r.top_labels) == len(r.top_log_probs) == 3 and r.log_prob is None
    want = ao.scores(StandIn().rows(v.volume), 1.5, top=3)
    assert r.top_labels[0].dtype == np.uint8 and r.entropy.dtype == np.float32
    assert np.array_equal(r.top_labels[1].volume.reshape(-1), want["top_label"][:, 1])
    assert np.allclose(r.entropy.volume.reshape(-1), want["entropy"], rtol=0, atol=1e-6)
    other = v.reformat(("AP", "LR", "SI"))
    r2 = m.generate_scores(other, top=3, temperature=1.5)
    for a, b in ((r.entropy, r2.entropy), (r.top_labels[2], r2.top_labels[2]), (r.top_log_probs[0], r2.top_log_probs[0])):
        assert b.orientation == other.orientation and np.allclose(b.affine, other.affine)
        assert np.array_equal(b.reformat(v.orientation).volume, a.volume)


@pytest.mark.parametrize("dtype", [np.uint8, np.int16, np.int64])
def test_given_labels_in_any_orientation_and_type(dtype):
    m, v = Model(), volume(1)
    lab = np.random.default_rng(2).integers(0, 5, (H, W, S)).astype(dtype)
    lab[0, 0] = 255 if dtype == np.uint8 else -1
    given = MedicalVolume(lab, AFFINE).reformat(("LR", "SI", "AP"))
    r = m.generate_scores(v, labels=given)
    want = ao.scores(StandIn().rows(v.volume), 1.0, lab.astype(np.int64).reshape(-1), ignore=255 if dtype == np.uint8 else -1)
    assert np.allclose(r.log_prob.volume.reshape(-1), want["log_prob"], rtol=0, atol=1e-6)
    assert np.all(r.log_prob.volume[0, 0] == 0)


def test_divergence_of_a_models_own_answers_is_zero():
    m, v = Model(), volume(3)
    r = m.generate_scores(v, top=2)
    d = m.divergence(v, r)
    assert d.dtype == np.float32 and d.shape == v.shape and np.abs(d.volume).max() < 1e-6  # (the stored values are rounded)
    far = MedicalVolume(v.volume + 1.0, AFFINE)
    assert m.divergence(far, r).volume.max() > 0.01
    axial = v.reformat(("AP", "LR", "SI"))
    d2 = m.divergence(axial, r)  # the answers are brought to the volume's voxels
    assert d2.orientation == axial.orientation and np.abs(d2.volume).max() < 1e-6


def test_label_map_feeds_to_metrics():
    from dosma_amd.quant_vals import T2

    m, v = Model(), volume(4)
    r = m.generate_scores(v)
    qv = T2(MedicalVolume(np.abs(v.volume) + 30.0, AFFINE))
    names = {i + 1: c for i, c in enumerate(m.CATEGORIES)}
    df = qv.to_metrics(r.top_labels[0], names, fns={"n": len})
    counts = np.bincount(r.top_labels[0].volume.reshape(-1), minlength=5)
    assert list(df["# Voxels"][:4]) == list(counts[1:5])


def test_refusals():
    m, v = Model(), volume(5)
    r = m.generate_scores(v)
    for call, says in (
            (lambda: m.generate_scores(v, top=0), "`top` must be"), (lambda: m.generate_scores(v, top=6), "`top` must be"),
            (lambda: m.generate_scores(v.volume), "3D MedicalVolume"),
            (lambda: m.generate_scores(MedicalVolume(np.zeros((H + 1, W, S), np.float32), AFFINE)), "built for slices"),
            (lambda: m.generate_scores(v, labels=v.volume), "must be a MedicalVolume"),
            (lambda: m.generate_scores(v, labels=v), "must be integers"),
            (lambda: m.generate_scores(v, labels=MedicalVolume(np.full((H, W, S), 300), AFFINE)), "255"),
            (lambda: m.generate_scores(v, labels=MedicalVolume(np.zeros((H, W, S + 1), np.uint8), AFFINE)), "has shape"),
            (lambda: m.divergence(v, AnswerMaps([], [], None, None)), "holds no labels"),
            (lambda: m.divergence(v, r._replace(top_log_probs=[])), "holds no labels")):
        with pytest.raises(ValueError, match=says):
            call()


def test_single_class_and_qdess_models_share_them():
    assert StanfordQDessUNet2D.generate_scores is OAIUnet2D.generate_scores
    m = object.__new__(StanfordQDessUNet2D)
    with pytest.raises(ValueError, match="3D or 4D"):
        m._single_volume(volume().volume)
    v = volume()
    assert m._single_volume(v) is v
