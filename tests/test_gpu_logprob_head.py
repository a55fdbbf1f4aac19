"""OutputHead.token_logprobs and OutputHead.distillation_loss on a B200: the fused node (RMSNorm -> FP8
lm_head -> soft cap -> operator) against the definitions in 64 bits on plainly computed logits of the same
fp8 recipe, and its gradients against a plain computation of the same recipe.

Tolerances.  The node's logits and the plain ones are one bf16 rounding of two f32 sums in different
orders (and a soft cap of three roundings): at most one bf16 step apart, which is 2^-4 for 8 <= |logit| <
16.  A log probability moves by at most |dx_t| + sum_v p_v |dx_v|, so by two steps: 2^-3.  Gradients go
through fp8 GEMMs: the tolerance of helpers.py against a reference that quantises the same way, with the
same scale (from the bound of |dl| that the rows' results allow).  The fp8 logit gradient itself is checked
on the kernels: half a step of the format."""
import pytest
import torch

from helpers import compare

pytestmark = pytest.mark.gpu
LOGIT = 2.0 ** -3


def make_head(cuda, d, V, cap, seed=0):
    from macrogpt_jax_b200.einsum import Rngs
    from macrogpt_jax_b200.head import OutputHead
    head = OutputHead(d, V, head_cap=cap, rngs=Rngs(seed))
    g = torch.Generator(device=cuda).manual_seed(seed)
    with torch.no_grad():
        head.lm_head.w.copy_(torch.randn((d, V), generator=g, device=cuda) * 3 * d ** -0.5)
        head.norm.scale.copy_(1 + 0.3 * torch.randn(d, generator=g, device=cuda))
    x = torch.randn((2, 48, d), generator=g, device=cuda).bfloat16()
    return head, x, g


def fp8(t, dt, fmax, amax=None):
    s = fmax / (t.abs().max().float().clamp(min=1e-30) if amax is None else amax)
    return (t.float() * s).to(dt).float() / s


def plain_operands(head, xn):
    return (fp8(xn.detach().bfloat16(), torch.float8_e4m3fn, 448.0),
            fp8(head.lm_head.w.detach(), torch.float8_e4m3fn, 448.0))


def capped(head, qx, qw):
    logits = (qx @ qw).bfloat16().float()
    if head.head_cap != "tanh":
        return logits
    return (15 * torch.tanh((logits / 15).bfloat16().float()).bfloat16().float()).bfloat16().float()


def plain_logits(head, x):
    x = x.detach().float()
    xn = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + head.norm.eps) * head.norm.scale.detach().float()
    return capped(head, *plain_operands(head, xn))


def head_reference(head, x, grad_logits, bound):
    """Gradients of sum(<grad_logits(logits), logits>) with the node's recipe: e4m3 operands, the logit
    gradient in the lm_head's bwd_dtype with the scale of `bound`, f32 products, the norm by autograd."""
    x = x.detach().float().requires_grad_(True)
    scale = head.norm.scale.detach().float().requires_grad_(True)
    xn = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + head.norm.eps) * scale
    qx, qw = plain_operands(head, xn)
    c = capped(head, qx, qw)
    dl = grad_logits(c)
    if head.head_cap == "tanh":
        dl = dl * (1 - (c / 15) ** 2)
    qd = fp8(dl, torch.float8_e5m2, 57344.0, bound)
    dw = qx.reshape(-1, qx.shape[-1]).T @ qd.reshape(-1, qd.shape[-1])
    dxn = (qd @ qw.T).bfloat16().float()
    dx, ds = torch.autograd.grad(xn, (x, scale), dxn)
    return dx, ds, dw


@pytest.mark.parametrize("cap,V", [(None, 1000), ("tanh", 1000), ("tanh", 2048)])
def test_head_scores(cuda, cap, V):
    head, x, g = make_head(cuda, 256, V, cap)
    tok = torch.randint(0, V, (2, 48), generator=g, device=cuda)
    mask = torch.rand((2, 48), generator=g, device=cuda) > 0.3
    with torch.no_grad():
        out = head.token_logprobs(x, tok, top_k=5, temperature=0.8, mask=mask)
        logits = plain_logits(head, x)
    assert logits.abs().max() < 16
    logp = torch.log_softmax(logits.double() / 0.8, -1)
    tol = LOGIT / 0.8
    ref = torch.where(mask, logp.gather(2, tok[..., None])[..., 0], 0.0)
    assert (out.logprob.double() - ref).abs().max() <= tol
    H = torch.where(mask, -(logp.exp() * logp).sum(-1), 0.0)
    # dH/dx_v = -p_v (log p_v + H): at most max(log V, H) in sum
    assert (out.entropy.double() - H).abs().max() <= tol * 8
    assert (out.top_ids[~mask] == -1).all()
    got = logp.gather(2, out.top_ids.clamp(min=0))
    best = logp.topk(5, dim=-1).values
    assert ((got - best).abs()[mask] <= tol).all()
    assert ((out.top_logprobs.double() - best).abs()[mask] <= tol).all()


@pytest.mark.parametrize("cap,V", [(None, 1000), ("tanh", 1000), ("tanh", 2048)])
def test_head_score_gradients(cuda, cap, V):
    head, x, g = make_head(cuda, 256, V, cap, 3)
    tok = torch.randint(0, V, (2, 48), generator=g, device=cuda)
    mask = torch.rand((2, 48), generator=g, device=cuda) > 0.3
    adv = torch.randn((2, 48), generator=g, device=cuda)
    x = x.requires_grad_(True)
    out = head.token_logprobs(x, tok, top_k=3, mask=mask)
    dtop = torch.randn(out.top_logprobs.shape, generator=g, device=cuda) * 0.1
    loss = (out.logprob * adv).sum() + 0.05 * out.entropy.sum() + (out.top_logprobs * dtop)[mask].sum()
    loss.backward()

    def grad(c):
        c = c.double().requires_grad_(True)
        lp = torch.log_softmax(c, -1)
        val = (lp.gather(2, tok[..., None])[..., 0] * adv - 0.05 * (lp.exp() * lp).sum(-1))[mask].sum()
        val = val + (lp.gather(2, out.top_ids.clamp(min=0)) * dtop)[mask].sum()
        return torch.autograd.grad(val, c)[0].float()

    bound = ((adv.abs() + 0.05 * (0.368 + out.entropy.detach()) + dtop.abs().sum(-1)) * mask).max()
    dx, ds, dw = head_reference(head, x, grad, bound)
    for a, b in ((x.grad, dx), (head.norm.scale.grad, ds), (head.lm_head.w.grad, dw)):
        compare(a.double().cpu().numpy(), b.double().cpu().numpy())


@pytest.mark.parametrize("cap,V,T", [(None, 1000, 1.0), ("tanh", 1000, 2.0), ("tanh", 2048, 1.0)])
def test_teacher_head_to_student_head(cuda, cap, V, T):
    """The distillation step as it is used: the teacher's head gives its top entries, the student's head
    the loss and the gradients."""
    teacher, x, g = make_head(cuda, 256, V, cap, 1)
    student = make_head(cuda, 256, V, cap, 2)[0]
    mask = torch.rand((2, 48), generator=g, device=cuda) > 0.2
    with torch.no_grad():
        top = teacher.token_logprobs(x, top_k=16, entropy=False, mask=mask)
    x = x.requires_grad_(True)
    loss = student.distillation_loss(x, top.top_ids, top.top_logprobs, temperature=T, mask=mask)
    assert loss.shape == (2, 48) and (loss[~mask] == 0).all()
    loss.sum().backward()
    ids = top.top_ids.clamp(min=0)
    q = torch.softmax(torch.where(mask[..., None], top.top_logprobs, 0.0).double() / T, -1)

    def value(c):
        lp = torch.log_softmax(c.double() / T, -1)
        return ((q * (q.log() - lp.gather(2, ids))).sum(-1) * mask)

    with torch.no_grad():
        logits = plain_logits(student, x)
        ref = value(logits)
    assert logits.abs().max() < 16
    assert (loss.double() - ref).abs().max() <= LOGIT / T

    def grad(c):
        c = c.double().requires_grad_(True)
        return torch.autograd.grad(value(c).sum(), c)[0].float()

    dx, ds, dw = head_reference(student, x, grad, torch.tensor(1 / T, device=cuda))
    for a, b in ((x.grad, dx), (student.norm.scale.grad, ds), (student.lm_head.w.grad, dw)):
        compare(a.double().cpu().numpy(), b.double().cpu().numpy())


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("cap", [0.0, 15.0])
def test_head_gradient_kernel(cuda, fmt, cap):
    """The gradient kernel's fp8 output (soft cap, padded pitch): dlogits against the formula, the scale from
    the rows' bound, zeros where every row is masked."""
    from macrogpt_jax_b200 import ops
    T, V, Vp = 37, 1000, 1008
    g = torch.Generator(device=cuda).manual_seed(7)
    c = (15 * torch.tanh(torch.randn((T, Vp), generator=g, device=cuda) / 3)).bfloat16()
    tok = torch.randint(0, V, (T,), generator=g, device=cuda)
    mask = torch.rand(T, generator=g, device=cuda) > 0.5
    adv = torch.randn(T, generator=g, device=cuda)
    lg = c[:, :V]
    out = ops.token_logprobs_forward(lg, tok, mask, 4, 1.0, True, True)
    ent, top_id, stats = out[1], out[3], out[4]
    dent = torch.full((T,), 0.1, device=cuda)
    dtop = torch.randn((T, 4), generator=g, device=cuda) * 0.1
    q = ops.token_logprobs_backward(lg, stats, tok, mask, 1.0, adv, dent, dtop, top_id, (cap, fmt, Vp))
    assert q.q.shape == (T, Vp)
    fmax, eps, tiny = ((448.0, 2.0 ** -3, 2.0 ** -9), (57344.0, 2.0 ** -2, 2.0 ** -16))[fmt]
    # the bound, and inv_scale = 1 / (fmax / amax): three roundings
    bound = ((adv.abs() + 0.1 * (0.368 + ent.abs()) + dtop.abs().sum(1)) * mask).double().max()
    assert abs(q.amax.item() - bound) <= 8 * 2.0 ** -24 * bound
    assert abs(q.inv_scale.item() - q.amax.item() / fmax) <= 3 * 2.0 ** -24 * q.amax.item() / fmax
    x = lg.double().requires_grad_(True)
    lp = torch.log_softmax(x, -1)
    val = lp.gather(1, tok[:, None])[:, 0] * adv + 0.1 * -(lp.exp() * lp).sum(-1)
    val = (val + (lp.gather(1, top_id.clamp(min=0)) * dtop).sum(-1))[mask].sum()
    ref, = torch.autograd.grad(val, x)
    ref = ref * (1 - (x.detach() / cap) ** 2) if cap else ref
    deq = q.q[:, :V].double() * q.inv_scale.double()
    # half a step of the format (relative, or of its subnormals), and f32 work on values below `bound`
    tol = eps / 2 * ref.abs() + tiny / 2 * q.inv_scale.double() + 200 * 2.0 ** -24 * bound
    assert ((deq - ref).abs() <= tol).all(), ((deq - ref).abs() / tol).max()
    assert ref.abs().max() <= bound
    none = torch.zeros(T, dtype=torch.bool, device=cuda)
    q = ops.token_logprobs_backward(lg, stats, tok, none, 1.0, adv, None, None, None, (cap, fmt, Vp))
    assert q.amax.item() == 0 and q.inv_scale.item() == 1 and not q.q[:, :V].view(torch.uint8).any()
    # distillation: the bound is the largest upstream gradient
    ids = torch.rand((T, V), generator=g, device=cuda).argsort(-1)[:, :9].contiguous()
    t = torch.randn((T, 9), generator=g, device=cuda)
    dstats = ops.distill_forward(lg, ids, t, mask, 2.0, True)[1]
    q = ops.distill_backward(lg, dstats, ids, t, mask, 2.0, adv, (cap, fmt, Vp))
    assert q.amax.item() == (adv.abs() * mask).max().item() * 0.5
    dense = torch.zeros((T, V), dtype=torch.float64, device=cuda).scatter_(1, ids, torch.softmax(t.double() / 2, -1))
    ref = (torch.softmax(lg.double() / 2, -1) - dense) * (adv.double() * mask / 2)[:, None]
    ref = ref * (1 - (lg.double() / cap) ** 2) if cap else ref
    deq = q.q[:, :V].double() * q.inv_scale.double()
    tol = eps / 2 * ref.abs() + tiny / 2 * q.inv_scale.double() + 200 * 2.0 ** -24 * q.amax.double()
    assert ((deq - ref).abs() <= tol).all()


def test_head_retained_graph_and_changed_inputs(cuda):
    """A second backward through a retained graph gives the same bits; a token changed in place after the
    forward is noticed."""
    head, x, g = make_head(cuda, 128, 512, "tanh", 5)
    tok = torch.randint(0, 512, (2, 48), generator=g, device=cuda)
    x = x.requires_grad_(True)
    out = head.token_logprobs(x, tok)
    a, = torch.autograd.grad(out.logprob.sum(), x, retain_graph=True)
    b, = torch.autograd.grad(out.logprob.sum(), x, retain_graph=True)
    assert torch.equal(a, b)
    tok.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.logprob.sum(), x)


def test_generic_head(cuda):
    """A head that is not fused (a norm without bf16 scale) takes the same calls."""
    head, x, g = make_head(cuda, 128, 512, "tanh", 6)
    head.norm.scale.data = head.norm.scale.data.float()
    assert not head.fused()
    tok = torch.randint(0, 512, (2, 48), generator=g, device=cuda)
    x = x.requires_grad_(True)
    out = head.token_logprobs(x, tok, top_k=4)
    ref = torch.log_softmax(head.get_logits(x).double(), -1)
    assert (out.logprob.double() - ref.gather(2, tok[..., None])[..., 0]).abs().max() <= 1e-4
    loss = head.distillation_loss(x, out.top_ids, out.top_logprobs.detach())
    (loss.sum() - out.logprob.sum()).backward()
    assert x.grad.isfinite().all() and head.lm_head.w.grad.isfinite().all()


def test_head_without_entries(cuda):
    """No teacher entries: every loss is 0 and so are the gradients, as without the head."""
    head, x, _ = make_head(cuda, 128, 512, "tanh", 9)
    x = x.requires_grad_(True)
    none = torch.empty((2, 48, 0), device=cuda)
    loss = head.distillation_loss(x, none.long(), none)
    assert loss.shape == (2, 48) and not loss.any()
    loss.sum().backward()
    assert not x.grad.any() and not head.lm_head.w.grad.any()


def test_head_without_rows(cuda):
    """No positions: empty results, and gradients of 0."""
    head, x, _ = make_head(cuda, 128, 512, "tanh", 10)
    x = x[:, :0].requires_grad_(True)
    ids = torch.empty((2, 0, 4), dtype=torch.int64, device=cuda)
    out = head.token_logprobs(x, ids[..., 0], top_k=3)
    loss = head.distillation_loss(x, ids, torch.empty((2, 0, 4), device=cuda))
    assert out.logprob.shape == out.entropy.shape == loss.shape == (2, 0) and out.top_ids.shape == (2, 0, 3)
    (loss.sum() + out.logprob.sum()).backward()
    assert x.grad.shape == x.shape and not head.lm_head.w.grad.any()


def test_head_backward_reads_the_saved_tensors(cuda):
    """The backward takes every input from autograd, so that saved-tensor hooks can move them: hooks that
    hand back other tokens, teacher ids and masks than were saved give those tensors' gradient."""
    head, x, g = make_head(cuda, 128, 512, "tanh", 11)
    tok, tok2 = torch.randint(0, 512, (2, 2, 48), generator=g, device=cuda)
    keep, keep2 = torch.rand((2, 2, 48), generator=g, device=cuda) > 0.3
    ids, ids2 = torch.randint(0, 512, (2, 2, 48, 4), generator=g, device=cuda)
    t, t2 = torch.randn((2, 2, 48, 4), generator=g, device=cuda)
    x = x.requires_grad_(True)
    swaps = {a.data_ptr(): b for a, b in ((tok, tok2), (keep, keep2), (ids, ids2), (t, t2))}

    def unpack(s):
        return swaps[s.data_ptr()].reshape(s.shape) if s.data_ptr() in swaps else s

    def score(tok, keep):
        return head.token_logprobs(x, tok, mask=keep, entropy=False).logprob

    want, = torch.autograd.grad(score(tok2, keep & keep2).sum(), x)
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s, unpack):
        # rows that were masked in the forward have no statistics
        keep2 &= keep
        got, = torch.autograd.grad(score(tok, keep).sum(), x)
    assert torch.equal(got, want)
    # the teacher's statistics are the forward's: other ids, the same values
    swaps.pop(t.data_ptr())
    want, = torch.autograd.grad(head.distillation_loss(x, ids2, t, mask=keep2).sum(), x)
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s, unpack):
        got, = torch.autograd.grad(head.distillation_loss(x, ids, t, mask=keep).sum(), x)
    assert torch.equal(got, want)
