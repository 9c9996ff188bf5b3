"""The 4-bit teacher and distillation from its top logits together, as a training run uses them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_quantised_teacher_to_student_gradient():
    """An image through the encoder in 4 bits, its features through a 4-bit classifier, the classifier's top logits as targets, a student's
    logits by ops.linear against them: the loss and the gradients of the student's weight and bias, against the formulas in 64 bits on the
    same logits."""
    from functools import partial
    from samnerf_amd import losses, ops
    from samnerf_amd.image_encoder import ImageEncoderViT
    torch.manual_seed(0)
    enc = ImageEncoderViT(img_size=224, patch_size=16, embed_dim=256, depth=2, num_heads=4, mlp_ratio=2.0, out_chans=64, qkv_bias=True,
                          norm_layer=partial(torch.nn.LayerNorm, eps=1e-6), use_rel_pos=True, window_size=5, global_attn_indexes=(1,))
    enc = enc.cuda().eval().set_linear_format("mxfp4")
    feats = enc(torch.randn((1, 3, 224, 224), device="cuda"))            # [1, 64, 14, 14]
    rows = feats.permute(0, 2, 3, 1).reshape(-1, 64)                     # a row per patch
    classes, k, T = 1003, 16, 2.0
    head = ops.quantize_mxfp4(torch.randn((classes, 64), device="cuda"))
    teacher = ops.linear_mxfp4(rows, head)                               # [196, 1003]
    target = ops.top_logits(teacher, k, temperature=T)
    assert torch.equal(target.logits, torch.gather(teacher, 1, target.ids.long()))
    ids = target.ids.clone()
    ids[::7] = -1                                                        # patches outside the image
    x = torch.randn((196, 48), device="cuda")
    w = (0.1 * torch.randn((classes, 48), device="cuda")).requires_grad_(True)
    b = torch.zeros((classes,), device="cuda", requires_grad=True)
    for with_rest in (True, False):
        loss_fn = losses.TopLogitsDistillLoss(temperature=T, weight=0.5, with_rest=with_rest)
        student = ops.linear(x, w, b)
        student.retain_grad()
        loss = loss_fn(student, (ids, target.logits, target.rest))
        w.grad = b.grad = None
        loss.backward()
        # 64 bits, on the student's own logits
        z = student.detach().cpu().double().requires_grad_(True)
        logq = torch.log_softmax(z / T, 1)
        on = (ids[:, 0] >= 0).cpu()
        place = target.ids.cpu().long()
        a = target.logits.cpu().double() / T
        if with_rest:
            a = torch.cat([a, target.rest.cpu().double()[:, None]], 1)
            other = torch.logsumexp(logq.scatter(1, place, -math.inf), 1, keepdim=True)
            lq = torch.cat([logq.gather(1, place), other], 1)
        else:
            lq = logq.gather(1, place)
        lp = torch.log_softmax(a, 1)
        want = 0.5 * T * T * ((lp.exp() * (lp - lq)).sum(1)[on]).mean()
        (dz,) = torch.autograd.grad(want, z)
        # logarithms of sums of 1003 terms and logits of up to 20 / T: 160 steps of 2^-24 of their size (20), as the loss' own tests derive
        assert abs(float(loss.detach()) - float(want)) <= 0.5 * T * T * 160 * 2.0 ** -24 * 20
        n = int(on.sum())
        part = 0.5 * T / n * (torch.exp(logq.detach()) + 1.0)
        assert bool(((student.grad.cpu().double() - dz).abs() <= part * 160 * 2.0 ** -24 * 20).all())
        # the layer's own backward on that gradient: 3-term bf16 split, 2^-16 a product
        dw, db = dz.t() @ x.cpu().double(), dz.sum(0)
        mag = dz.abs().t() @ x.cpu().double().abs()
        assert bool(((w.grad.cpu().double() - dw).abs() <= 2.0 ** -14 * mag + 1e-9).all())
        assert bool(((b.grad.cpu().double() - db).abs() <= 2.0 ** -14 * dz.abs().sum(0) + 1e-9).all())
