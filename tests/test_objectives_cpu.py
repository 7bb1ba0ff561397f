"""Token objectives without a GPU: every refusal (Python and C ABI), the oracle against torch, the teacher's columns through
the feature cache's files and the collator."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import objectives as O
from speech_to_text_amd import _lib, distillation_loss, distillation_loss_and_grad, token_logprobs
from speech_to_text_amd.config import DataConfig
from speech_to_text_amd.data import AudioCollator
from speech_to_text_amd.feature_cache import FeatureCacheDataset, FeatureCacheWriter

Z = torch.zeros(2, 3, 11)
Y = torch.zeros(2, 3, dtype=torch.long)
IDS, T = torch.zeros(2, 3, 4, dtype=torch.long), torch.zeros(2, 3, 4)


@pytest.mark.parametrize("match, call", [
    ("float32, float16 or bfloat16", lambda: token_logprobs(Z.double(), Y)),
    ("has to be contiguous", lambda: token_logprobs(Z.transpose(1, 2), torch.zeros(2, 11, dtype=torch.long))),
    ("more than two row strides", lambda: token_logprobs(torch.zeros(4, 5, 6, 7)[::2, ::2, ::2], torch.zeros(2, 3, 3).long())),
    ("empty vocabulary", lambda: token_logprobs(torch.zeros(3, 0), torch.zeros(3).long())),
    ("tensor", lambda: token_logprobs(np.zeros((2, 3)), Y)),
    ("labels has shape", lambda: token_logprobs(Z, Y[:, :2])),
    ("labels is an int64", lambda: token_logprobs(Z, Y.float())),
    ("top_k", lambda: token_logprobs(Z, Y, top_k=12)),
    ("top_k", lambda: token_logprobs(torch.zeros(2, 100), top_k=65)),
    ("top_k", lambda: token_logprobs(Z, Y, top_k=-1)),
    ("nothing is asked for", lambda: token_logprobs(Z)),
    ("temperature", lambda: token_logprobs(Z, Y, temperature=0.0)),
    ("temperature", lambda: token_logprobs(Z, Y, temperature=float("nan"))),
    ("alpha", lambda: distillation_loss(Z, Y, IDS, T, alpha=1.5)),
    ("alpha", lambda: distillation_loss(Z, Y, IDS, T, alpha=float("nan"))),
    ("reduction", lambda: distillation_loss(Z, Y, IDS, T, reduction="batchmean")),
    ("weight", lambda: distillation_loss(Z, Y, IDS, T, reduction="none", weight=0.5)),
    ("temperature", lambda: distillation_loss(Z, Y, IDS, T, temperature=-1.0)),
    ("teacher_ids", lambda: distillation_loss(Z, Y, IDS[..., :0], T[..., :0])),
    ("teacher_ids", lambda: distillation_loss(Z, Y, torch.zeros(2, 3, 65).long(), torch.zeros(2, 3, 65))),
    ("teacher_ids", lambda: distillation_loss(Z, Y, IDS[0], T[0])),
    ("teacher_ids", lambda: distillation_loss(Z, Y, IDS.float(), T)),
    ("teacher_logits", lambda: distillation_loss(Z, Y, IDS, T[..., :3])),
    ("teacher_logits", lambda: distillation_loss(Z, Y, IDS, IDS)),
    ("no gradient here", lambda: distillation_loss(Z, Y, IDS, T.clone().requires_grad_())),
    ("reduction", lambda: distillation_loss_and_grad(Z, Y, IDS, T, reduction="none")),
])
def test_refusals(match, call):
    with pytest.raises(ValueError, match=match):
        call()


def test_no_cpu_path():
    with pytest.raises(_lib.SttfeError, match="no CPU path"):
        token_logprobs(Z, Y)
    with pytest.raises(_lib.SttfeError, match="no CPU path"):
        distillation_loss(Z, Y, IDS, T)


def test_c_abi_checks_arguments_before_the_gpu():
    L = _lib.lib()
    n = ctypes.c_size_t()
    p = ctypes.c_void_p(64)                    # never dereferenced: every call below is refused or has no rows

    def score(logits=p, dtype=0, outer=2, inner=3, so=33, si=11, V=11, labels=p, temp=1.0, k=0, lp=p, ids=None, top=None):
        return L.sttfe_token_logprobs(logits, dtype, outer, inner, so, si, V, labels, -100, temp, k, lp, None, None, ids, top,
                                      None, 0, None)

    assert score(outer=0) == 0 and score(inner=0) == 0
    assert score(logits=None) == -1 and score(dtype=3) == -1 and score(outer=-1) == -1 and score(so=-1) == -1
    assert score(V=0) == -1 and score(labels=None) == -1 and score(temp=0.0) == -1 and score(temp=float("inf")) == -1
    assert score(k=4) == -1 and score(k=12, ids=p, top=p) == -1 and score(k=65, V=100, ids=p, top=p) == -1
    assert score(logits=ctypes.c_void_p(66)) == -1                       # float32 at half an element
    assert score(outer=2 ** 40, inner=2 ** 40) == -5 and score(V=2 ** 22 + 1) == -5
    assert L.sttfe_token_logprobs_workspace_bytes(-1, 11, 0, 0, ctypes.byref(n)) == -1
    assert L.sttfe_token_logprobs_workspace_bytes(6, 11, 0, 12, ctypes.byref(n)) == -1
    assert L.sttfe_token_logprobs_workspace_bytes(6, 11, 0, 4, None) == -1
    assert L.sttfe_token_logprobs_workspace_bytes(6, 11, 0, 4, ctypes.byref(n)) == 0

    def grad(stats=p, out=p, gl=p, labels=p, k=0, ids=None, gt=None, outer=2):
        return L.sttfe_token_logprobs_grad(p, 0, outer, 3, 33, 11, 11, labels, -100, 1.0, stats, gl, None, k, ids, gt, out, None)

    assert grad(outer=0) == 0 and grad(stats=None) == -1 and grad(out=None) == -1 and grad(labels=None) == -1
    assert grad(gt=p) == -1 and grad(gt=p, k=3) == -1

    def distill(K=4, tau=1.0, alpha=0.5, red=2, losses=p, total=p, factor=p, labels=p, ids=p, t=p, outer=2):
        return L.sttfe_distill_loss(p, 2, outer, 3, 33, 11, 11, labels, -100, ids, t, K, tau, alpha, 1.0, red, losses, total, factor,
                                    None, None, None, 0, None)

    assert distill(outer=0, red=0) == 0
    assert distill(K=0) == -1 and distill(K=65) == -1 and distill(tau=0.0) == -1 and distill(alpha=-0.1) == -1
    assert distill(alpha=float("nan")) == -1 and distill(red=3) == -1 and distill(total=None) == -1 and distill(factor=None) == -1
    assert distill(losses=None) == -1 and distill(labels=None) == -1 and distill(ids=None) == -1 and distill(t=None) == -1
    assert L.sttfe_distill_workspace_bytes(6, 0, 0, ctypes.byref(n)) == -1
    assert L.sttfe_distill_grad(p, 2, 2, 3, 33, 11, 11, p, -100, p, p, 4, 1.0, 0.5, None, None, None, None, p, None) == -1
    assert L.sttfe_distill_grad(p, 2, 0, 3, 33, 11, 11, p, -100, p, p, 4, 1.0, 0.5, None, None, None, None, p, None) == 0
    assert L.sttfe_distill_rescale(p, 5, 3, p, None) == -1 and L.sttfe_distill_rescale(p, 0, -1, p, None) == -1
    assert L.sttfe_distill_rescale(None, 0, 3, p, None) == -1 and L.sttfe_distill_rescale(None, 0, 0, None, None) == 0


def test_oracle_against_torch_autograd():
    """The oracle's closed-form gradients equal torch's autograd of the definitions, in float64 (products of a handful of
    terms: 1e-13)."""
    g = torch.Generator().manual_seed(1)
    z = (3 * torch.randn(5, 23, generator=g, dtype=torch.float64)).requires_grad_()
    y = torch.tensor([3, -100, 0, 22, 7])
    ids = torch.tensor([[3, 1, 3], [2, 2, 2], [-1, 5, 6], [-1, -1, -1], [7, 9, 0]])
    t = torch.randn(5, 3, generator=g, dtype=torch.float64)
    tau, alpha, live = 1.7, 0.6, y >= 0
    lp, lp1 = torch.log_softmax(z / tau, 1), torch.log_softmax(z, 1)
    q = torch.nan_to_num(torch.softmax((t / tau).masked_fill(ids < 0, -torch.inf), 1))
    kl = (torch.xlogy(q, q) - q * lp.gather(1, ids.clamp_min(0))).sum(1)
    each = torch.where(live, alpha * tau ** 2 * kl - (1 - alpha) * lp1.gather(1, y.clamp_min(0)[:, None])[:, 0], 0.0)
    d, = torch.autograd.grad(each.sum(), z, retain_graph=True)
    loss, grad, _ = O.distillation(z.detach().numpy(), y.numpy(), ids.numpy(), t.numpy(), tau, alpha)
    assert np.abs(loss - each.detach().numpy()).max() < 1e-13 and np.abs(grad - d.numpy()).max() < 1e-13
    ent = -(lp.exp() * lp).sum(1)
    gl, gh, gt = torch.randn(5, generator=g).double(), torch.randn(5, generator=g).double(), torch.randn(5, 4, generator=g).double()
    top = lp.topk(4, 1)
    out = (gl * lp.gather(1, y.clamp_min(0)[:, None])[:, 0] + gh * ent + (gt * top.values).sum(1)) * live
    d, = torch.autograd.grad(out.sum(), z)
    grad, _ = O.token_logprobs_grad(z.detach().numpy(), y.numpy(), gl.numpy(), gh.numpy(), top.indices.numpy(), gt.numpy(), tau)
    assert np.abs(grad - d.numpy()).max() < 1e-13
    s = O.token_logprobs(z.detach().numpy(), y.numpy(), 4, tau)
    assert np.abs(s[1] - (ent * live).detach().numpy()).max() < 1e-13
    assert np.array_equal(s[2][live.numpy()], top.indices[live].numpy())


def test_oracle_order_of_alternatives():
    z = np.array([1.0, np.nan, -0.0, 5.0, 0.0, 5.0, -np.inf, np.inf])
    assert O.alternatives(z, 8).tolist() == [1, 7, 3, 5, 0, 2, 4, 6]


def _write(tmp_path, monkeypatch, teacher):
    """A cache of three clips, two batches; the GPU's answer is planted (token_logprobs has its own tests)."""
    from speech_to_text_amd import objectives
    seen = []

    def fake(logits, labels, top_k=0, **kw):
        seen.append((labels.tolist(), top_k))
        lp = torch.log_softmax(logits.float(), -1)
        v, i = lp.topk(top_k, -1)
        live = (labels != -100)[..., None]
        return objectives.TokenScores(None, None, torch.where(live, i, -1), torch.where(live, v, -torch.inf))

    monkeypatch.setattr(objectives, "token_logprobs", fake)
    w = FeatureCacheWriter(str(tmp_path), "speech2text", 8, shard_clips=2, teacher_top=3)
    g = torch.Generator().manual_seed(5)
    feats = torch.randn(3, 8, 20, generator=g)
    logits = torch.randn(3, 4, 17, generator=g)
    labels = [[5, 6], [], [1, 2, 3, 4]]
    w.add_batch([0, 1], feats[:2], [0, 0], labels=labels[:2], teacher_logits=logits[:2, :3] if teacher[0] else None)
    w.add_batch([2], feats[2:], [0], labels=labels[2:], teacher_logits=logits[2:] if teacher[1] else None)
    w.close()
    return FeatureCacheDataset(str(tmp_path)), logits, seen


def test_teacher_through_cache_and_collator(tmp_path, monkeypatch):
    ds, logits, seen = _write(tmp_path, monkeypatch, (True, True))
    assert seen == [([[0, 0, -100], [-100, -100, -100]], 3), ([[0, 0, 0, 0]], 3)]     # positions without a label are not read
    lp = torch.log_softmax(logits, -1)
    for clip, n in ((0, 2), (1, 0), (2, 4)):
        v, i = lp[clip, :n].topk(3, -1)
        assert torch.equal(ds[clip]["teacher_ids"], i) and torch.equal(ds[clip]["teacher_logits"], v)
    batch = AudioCollator(DataConfig(), "speech2text", True)([ds[2], None, ds[0], ds[1]])
    assert batch["teacher_ids"].shape == (3, 4, 3) and batch["teacher_ids"].dtype == torch.int64
    assert batch["labels"].tolist() == [[1, 2, 3, 4], [5, 6, -100, -100], [-100] * 4]
    assert torch.equal(batch["teacher_ids"][0], ds[2]["teacher_ids"]) and torch.equal(batch["teacher_logits"][1, :2], ds[0]["teacher_logits"])
    assert (batch["teacher_ids"][1, 2:] == -1).all() and (batch["teacher_logits"][2] == -torch.inf).all()


def test_cache_without_or_with_some_teachers(tmp_path, monkeypatch):
    ds, _, _ = _write(tmp_path / "none", monkeypatch, (False, False))
    assert "teacher_ids" not in ds[0] and not list((tmp_path / "none").glob("teacher*"))
    batch = AudioCollator(DataConfig(), "speech2text", True)([ds[0], ds[2]])
    assert "teacher_ids" not in batch
    ds, _, _ = _write(tmp_path / "some", monkeypatch, (False, True))
    assert "teacher_ids" not in ds[0] and ds[2]["teacher_ids"].shape == (4, 3)
    batch = AudioCollator(DataConfig(), "speech2text", True)([ds[0], ds[2]])
    assert (batch["teacher_ids"][0] == -1).all() and torch.equal(batch["teacher_ids"][1], ds[2]["teacher_ids"])


def test_teacher_refusals(tmp_path):
    w = FeatureCacheWriter(str(tmp_path), "speech2text", 8)
    f = torch.zeros(2, 8, 5)
    with pytest.raises(ValueError, match="labels of every clip"):
        w.add_batch([0, 1], f, [0, 0], teacher_logits=torch.zeros(2, 3, 9))
    with pytest.raises(ValueError, match="batch, positions, vocabulary"):
        w.add_batch([0, 1], f, [0, 0], labels=[[1], [2]], teacher_logits=torch.zeros(3, 3, 9))
    with pytest.raises(ValueError, match="longest clip has 4 labels"):
        w.add_batch([0, 1], f, [0, 0], labels=[[1], [2, 3, 4, 5]], teacher_logits=torch.zeros(2, 3, 9))
    with pytest.raises(ValueError, match="teacher_top"):
        FeatureCacheWriter(str(tmp_path), "whisper", 80, teacher_top=65)
    assert w.shards == []                      # a refused batch leaves nothing behind
    w.close()


def test_c_abi_refuses_unaligned_statistics_and_temperatures_out_of_range():
    L = _lib.lib()
    p, odd = ctypes.c_void_p(64), ctypes.c_void_p(72)      # never dereferenced: every call below is refused

    def score(stats=None, ws=None, temp=1.0):
        return L.sttfe_token_logprobs(p, 0, 2, 3, 33, 11, 11, p, -100, temp, 0, p, None, stats, None, None, ws, 0, None)

    def grad(stats=p, temp=1.0):
        return L.sttfe_token_logprobs_grad(p, 0, 2, 3, 33, 11, 11, p, -100, temp, stats, p, None, 0, None, None, p, None)

    def distill(stats=None, ws=None, temp=1.0):
        return L.sttfe_distill_loss(p, 2, 2, 3, 33, 11, 11, p, -100, p, p, 4, temp, 0.5, 1.0, 2, p, p, p, stats, None, ws, 0, None)

    def distill_grad(stats=p, temp=1.0):
        return L.sttfe_distill_grad(p, 2, 2, 3, 33, 11, 11, p, -100, p, p, 4, temp, 0.5, stats, None, None, None, p, None)

    for call in (score, grad, distill, distill_grad):
        assert call(stats=odd) == -1
        for temp in (1e-7, 1e7, -1.0, float("nan"), float("inf")):
            assert call(temp=temp) == -1
    assert score(ws=odd) == -1 and distill(ws=odd) == -1


def test_workspace_queries_know_the_limits():
    L, n = _lib.lib(), ctypes.c_size_t()
    for rows, V in ((2 ** 24 + 1, 11), (6, 2 ** 21 + 1), (6, 2 ** 31 - 1), (2 ** 62, 2 ** 31 - 1)):
        assert L.sttfe_token_logprobs_workspace_bytes(rows, V, 0, 4, ctypes.byref(n)) == -5
        assert L.sttfe_distill_workspace_bytes(rows, V, 0, ctypes.byref(n)) == -5
    for dtype, e in ((0, 4), (1, 2), (2, 2)):
        assert L.sttfe_token_logprobs_workspace_bytes(2 ** 24, 2 ** 21, dtype, 64, ctypes.byref(n)) == 0
        assert n.value >= 2 ** 24 * (2 ** 21 * e // (2 ** 17)) * (16 + 8 * 64)


@pytest.mark.parametrize("call", [
    lambda z, t: token_logprobs(z, Y, entropy=True),
    lambda z, t: distillation_loss(z, Y, IDS, t),
    lambda z, t: distillation_loss(Z, Y, IDS, t + 0 * z[..., :4]),
    lambda z, t: distillation_loss_and_grad(z, Y, IDS, t),
])
def test_forward_mode_tangents_are_refused(call):
    """A dual tensor does not require a gradient: its tangent would be lost without a word."""
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode tangent"):
            call(forward_ad.make_dual(Z, torch.ones_like(Z)), T)
        with pytest.raises(_lib.SttfeError, match="no CPU path"):
            call(Z, T)


@pytest.mark.parametrize("scale", [torch.ones(2), torch.ones((), dtype=torch.float64), torch.ones((), dtype=torch.int64),
                                   torch.ones((), device="meta")])
def test_refused_scales_of_a_gradient(scale):
    with pytest.raises(ValueError, match="grad_scale"):
        distillation_loss_and_grad(Z, Y, IDS, T, grad_scale=scale)


def test_forward_mode_tangent_of_a_scale_is_refused():
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        scale = forward_ad.make_dual(torch.ones(()), torch.ones(()))
        with pytest.raises(ValueError, match="forward-mode tangent"):
            distillation_loss_and_grad(Z, Y, IDS, T, grad_scale=scale)
        with pytest.raises(_lib.SttfeError, match="no CPU path"):
            distillation_loss_and_grad(Z, Y, IDS, T, grad_scale=torch.ones(()))
