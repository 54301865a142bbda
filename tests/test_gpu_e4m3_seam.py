"""The 8-bit layers of a training pass are the call's own choice: an update() with dense="e4m3" leaves the heads that it used as they were."""
import pytest
import torch

from tests.test_gpu_e4m3_nodes import _train_model, _Trainer

pytestmark = pytest.mark.gpu


def _counted(monkeypatch):
    from phonlp_amd import ops
    calls = []
    plain = ops.linear_e4m3
    monkeypatch.setattr(ops, "linear_e4m3", lambda *a, **k: calls.append(1) or plain(*a, **k))
    return calls


def test_an_8_bit_update_leaves_the_heads_as_they_were(golden, monkeypatch):
    """Direct losses with masks on the trainer's own heads, with no parameter changed in between, are the fp32 ones before and after."""
    from phonlp_amd import compat
    z = golden("trainer_small.npz")
    T = lambda k: torch.from_numpy(z[k])
    batches = ((T("dep_tokens"), T("dep_first"), T("dep_mask"), T("loss_gold_head"), T("dep_gold_rel"), int(z["dep_nwords"]),
                z["dep_oidx"].tolist(), z["dep_lens"].tolist()),
               (T("tag_tokens"), T("tag_first"), T("gold_upos"), z["tag_oidx"].tolist(), z["tag_lens"].tolist()),
               (T("tag_tokens"), T("tag_first"), T("tag_mask"), T("gold_ner"), z["tag_oidx"].tolist(), z["tag_lens"].tolist()))
    calls = _counted(monkeypatch)
    model = _train_model(z)
    params = {k: v for k, v in model._heads.items() if v.requires_grad}
    lens = z["tag_lens"].tolist()

    def losses(**kw):
        heads = compat.refresh_heads(model)
        with torch.no_grad():
            enc = compat._encode_train(model.eval(), T("tag_tokens"), T("tag_first"))
        B, L = enc.shape[:2]
        drawn = lambda task: compat.draw_masks(heads, task, B, L, lens, 0.0, 0.0, enc.device)
        return (compat.pos_loss(heads, params, enc, lens, T("gold_upos"), masks=drawn("pos"), **kw).item(),
                compat.ner_loss(heads, params, enc, lens, T("gold_ner"), drawn("ner"), **kw).item())

    before = losses()
    assert not calls
    compat.patch_trainer(_Trainer(model), move_encoder=False, train_seam=True, dense="e4m3").update(*batches, 0.4, 0.2, 0.4)
    n = len(calls)
    assert n >= 6
    assert losses() == before and len(calls) == n
    assert losses(dense="e4m3") != before and len(calls) == n + 2
    assert losses(dense="f32") == before and len(calls) == n + 2


def test_refusals(golden):
    from phonlp_amd import compat
    z = golden("trainer_small.npz")
    model = _train_model(z)
    heads = compat.refresh_heads(model)
    enc = torch.zeros(2, 5, heads.w.upos_hid_w.shape[1], device=heads.w.trans.device)
    with pytest.raises(ValueError, match="dense"):
        heads.pos_backward(enc, [3, 5], torch.zeros(2, 5), dense="e5m2")
    for f, gold in ((heads.pos_backward, (torch.zeros(2, 5),)), (heads.ner_backward, (torch.zeros(2, 5),)),
                    (heads.parser_backward, (torch.zeros(2, 4), torch.zeros(2, 4)))):
        with pytest.raises(ValueError, match="masks"):
            f(enc, [3, 5], *gold, dense="e4m3")
