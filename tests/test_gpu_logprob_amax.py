"""The output head's logit gradient as fp8 with the scale of its largest value (AMAX_EXACT, what a head with an
e4m3 bwd_dtype takes), on a B200 against the formulas in 64 bits."""
import pytest
import torch

from helpers import compare
from test_gpu_logprob_head import capped, plain_logits

pytestmark = pytest.mark.gpu


def fp8(t, dt):
    """t as fp8 with the scale FMAX / amax.  A tensor over a tensor: torch takes a number over a tensor as the
    number times its reciprocal, one step of f32 off, and then a product such as 448 / 4.3125 * 1.6171875 =
    168, half way between two codes, goes the other way."""
    s = torch.full((), torch.finfo(dt).max, device=t.device) / t.abs().max().float()
    return (t.float() * s).to(dt).float() / s


def score_ref(c, tok, mask, adv, dent, dtop, top_id, cap):
    """Gradient of the rows' results at the capped logits c, before the cap, in 64 bits."""
    x = c.double().requires_grad_(True)
    lp = torch.log_softmax(x, -1)
    val = lp.gather(1, tok[:, None])[:, 0] * adv - dent * (lp.exp() * lp).sum(-1)
    val = (val + (lp.gather(1, top_id.clamp(min=0)) * dtop).sum(-1))[mask].sum()
    ref, = torch.autograd.grad(val, x)
    return ref * (1 - (x.detach() / cap) ** 2) if cap else ref


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("cap", [0.0, 15.0])
@pytest.mark.parametrize("T,V", [(37, 1000), (3, 9), (5, 40003)])
def test_exact_amax(cuda, fmt, cap, T, V):
    """AMAX_EXACT: the scale is that of the largest |dlogits|, and every value is within half a step of the
    format under it."""
    from macrogpt_jax_b200 import _capi as C
    from macrogpt_jax_b200 import ops
    Vp = (V + 15) // 16 * 16
    g = torch.Generator(device=cuda).manual_seed(V)
    c = (15 * torch.tanh(torch.randn((T, Vp), generator=g, device=cuda) / 3)).bfloat16()
    c[:, V:] = float("nan")  # columns past the last one are not read
    tok = torch.randint(0, V, (T,), generator=g, device=cuda)
    mask = torch.rand(T, generator=g, device=cuda) > 0.3
    mask[0] = True
    adv, dent = torch.randn((2, T), generator=g, device=cuda)
    dtop = torch.randn((T, 4), generator=g, device=cuda) * 0.1
    lg, head = c[:, :V], (cap, fmt | C.AMAX_EXACT, Vp)
    out = ops.token_logprobs_forward(lg, tok, mask, 4, 1.0, True, True)
    q = ops.token_logprobs_backward(lg, out[4], tok, mask, 1.0, adv, dent, dtop, out[3], head)
    ref = score_ref(lg, tok, mask, adv, dent, dtop, out[3], cap)
    fmax, eps, tiny = ((448.0, 2.0 ** -3, 2.0 ** -9), (57344.0, 2.0 ** -2, 2.0 ** -16))[fmt]
    # f32 work on terms of at most this size
    f32 = 200 * 2.0 ** -24 * ((adv.abs() + dent.abs() * (1 + out[1]) + dtop.abs().sum(1)) * mask).double().max()

    def check(q, ref, f32):
        amax = ref.abs().max()
        assert abs(q.amax.item() - amax) <= f32
        assert abs(q.inv_scale.item() - q.amax.item() / fmax) <= 3 * 2.0 ** -24 * q.amax.item() / fmax
        deq = q.q[:, :V].double() * q.inv_scale.double()
        assert ((deq - ref).abs() <= eps / 2 * ref.abs() + tiny / 2 * q.inv_scale.double() + f32).all()
        assert q.q[:, :V].float().abs().max() == fmax  # the largest value takes the largest code

    check(q, ref, f32)
    none = torch.zeros(T, dtype=torch.bool, device=cuda)
    q = ops.token_logprobs_backward(lg, out[4], tok, none, 1.0, adv, None, None, None, head)
    assert q.amax.item() == 0 and q.inv_scale.item() == 1 and not q.q[:, :V].view(torch.uint8).any()
    ids = torch.rand((T, V), generator=g, device=cuda).argsort(-1)[:, :9].contiguous()
    t = torch.randn((T, 9), generator=g, device=cuda)
    dstats = ops.distill_forward(lg, ids, t, mask, 2.0, True)[1]
    q = ops.distill_backward(lg, dstats, ids, t, mask, 2.0, adv, head)
    dense = torch.zeros((T, V), dtype=torch.float64, device=cuda).scatter_(1, ids, torch.softmax(t.double() / 2, -1))
    ref = (torch.softmax(lg.double() / 2, -1) - dense) * (adv.double() * mask / 2)[:, None]
    check(q, ref * (1 - (lg.double() / cap) ** 2) if cap else ref, f32)
    bad = adv.clone()
    bad[0] = float("nan")
    q = ops.distill_backward(lg, dstats, ids, t, mask, 2.0, bad, head)
    assert q.amax.isnan().all() and q.inv_scale.isnan().all()


def test_exact_amax_of_certain_rows(cuda):
    """Rows that are all but certain of their token: what is left is rounding in part, and no code is NaN
    or past the largest, whichever way the last unit of an odd row is stored."""
    from macrogpt_jax_b200 import _capi as C
    from macrogpt_jax_b200 import ops
    for V in (1001, 1003, 1007):
        c = torch.zeros((64, V + 1), dtype=torch.bfloat16, device=cuda)[:, :V]
        tok = torch.full((64,), V - 1, device=cuda)
        c[:, -1] = torch.linspace(20.5, 24, 64, device=cuda)
        out = ops.token_logprobs_forward(c, tok, None, 0, 1.0, True, True)
        adv = torch.linspace(1, 3, 64, device=cuda)
        q = ops.token_logprobs_backward(c, out[4], tok, None, 1.0, adv, None, None, None, (0.0, C.AMAX_EXACT, 1008))
        codes = q.q[:, :V].float()
        assert codes.isfinite().all() and codes.abs().max() == 448


def test_e4m3_entropy_gradient_of_a_large_vocabulary(cuda):
    """A flat row's entropy gradient is some thousand times below the bound from the rows' results.  With the
    scale of its largest value e4m3 loses what it has to: half a step of each value, 2^-4 of it, and half a
    subnormal step, 2^-10 / 448 of the largest, where values are smaller than that."""
    from macrogpt_jax_b200 import _capi as C
    from macrogpt_jax_b200 import ops
    T, V = 4, 128256
    g = torch.Generator(device=cuda).manual_seed(2)
    c = torch.randn((T, V), generator=g, device=cuda).bfloat16()
    out = ops.token_logprobs_forward(c, None, None, 0, 1.0, True, True)
    dent = torch.ones(T, device=cuda)
    q = ops.token_logprobs_backward(c, out[4], None, None, 1.0, None, dent, None, None, (0.0, C.AMAX_EXACT, V))
    lp = torch.log_softmax(c.double(), -1)
    H = -(lp.exp() * lp).sum(-1, keepdim=True)
    ref = -lp.exp() * (lp + H)
    # f32: p good to the row's sums (V / 2048 + 73 roundings) and a few more of log p
    f32 = 2.0 ** -24 * (V // 2048 + 100) * (lp.exp() * (lp.abs() + H)).norm()
    tol = 2.0 ** -4 * ref.norm() + (T * V) ** 0.5 * 2.0 ** -10 / 448 * ref.abs().max() + f32
    err = (q.q.double() * q.inv_scale.double() - ref).norm()
    assert err <= tol, (err / ref.norm(), tol / ref.norm())
    # only values below half a subnormal step (or f32's error) are lost
    lost = q.q.float() == 0
    f32 = 2.0 ** -24 * (V // 2048 + 100) * lp.exp() * (lp.abs() + H)
    assert (ref.abs() <= 1.001 * 2.0 ** -10 / 448 * ref.abs().max() + f32)[lost].all()


@pytest.mark.parametrize("cap,V", [(None, 1000), ("tanh", 32768)])
@pytest.mark.parametrize("kind", ["entropy", "near_teacher"])
def test_e4m3_head_gradients(cuda, cap, V, kind):
    """A head whose lm_head has an e4m3 bwd_dtype, on rows whose gradient is far below what the rows' results
    allow: its gradients are those of the same recipe with the scale of the largest logit gradient."""
    from macrogpt_jax_b200.einsum import Einsum, Rngs
    from macrogpt_jax_b200.head import OutputHead
    head = OutputHead(256, V, head_cap=cap, lm_head=Einsum.override(bwd_dtype=torch.float8_e4m3fn), rngs=Rngs(0))
    g = torch.Generator(device=cuda).manual_seed(V)
    with torch.no_grad():
        head.lm_head.w.copy_(torch.randn((256, V), generator=g, device=cuda) / 16)
        head.norm.scale.fill_(1.0)
    x = torch.randn((2, 48, 256), generator=g, device=cuda).bfloat16()
    logits = plain_logits(head, x)
    top = logits.topk(64, dim=-1)
    teacher = (top.values + 0.01 * torch.randn((2, 48, 64), generator=g, device=cuda)).contiguous()
    q = torch.softmax(teacher.double(), -1)
    x = x.requires_grad_(True)
    if kind == "entropy":
        head.token_logprobs(x).entropy.sum().backward()
    else:
        head.distillation_loss(x, top.indices, teacher).sum().backward()

    def grad(c):
        lp = torch.log_softmax(c.double(), -1)
        if kind == "entropy":
            return (-lp.exp() * (lp - (lp.exp() * lp).sum(-1, keepdim=True))).float()
        return lp.exp().scatter_add_(2, top.indices, -q).float()

    xr = x.detach().float().requires_grad_(True)
    scale = head.norm.scale.detach().float().requires_grad_(True)
    xn = xr * torch.rsqrt(xr.square().mean(-1, keepdim=True) + head.norm.eps) * scale
    qx = fp8(xn.detach().bfloat16(), torch.float8_e4m3fn)
    qw = fp8(head.lm_head.w.detach(), torch.float8_e4m3fn)
    c = capped(head, qx, qw)
    dl = grad(c)
    dl = fp8(dl * (1 - (c / 15) ** 2) if cap else dl, torch.float8_e4m3fn)
    dx, ds = torch.autograd.grad(xn, (xr, scale), (dl @ qw.T).bfloat16().float())
    dw = qx.reshape(-1, 256).T @ dl.reshape(-1, V)
    for a, b in ((x.grad, dx), (head.norm.scale.grad, ds), (head.lm_head.w.grad, dw)):
        compare(a.double().cpu().numpy(), b.double().cpu().numpy())


@pytest.mark.parametrize("fmt", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_head_step_replayed(cuda, fmt):
    """The head's operators, forward and backward, captured and replayed on new inputs and run on another
    stream: the same bits.  A larger gradient first, so that a stale largest value would show."""
    from macrogpt_jax_b200.einsum import Einsum, Rngs
    from macrogpt_jax_b200.graphs import GraphedStep
    from macrogpt_jax_b200.head import OutputHead
    head = OutputHead(128, 1000, lm_head=Einsum.override(bwd_dtype=fmt), rngs=Rngs(0))
    g = torch.Generator(device=cuda).manual_seed(4)
    with torch.no_grad():
        head.lm_head.w.copy_(torch.randn((128, 1000), generator=g, device=cuda) / 11)
    w = head.lm_head.w

    def step(x, tok, ids, t, up):
        x = x.detach().requires_grad_(True)
        out = head.token_logprobs(x, tok, top_k=4)
        loss = head.distillation_loss(x, ids, t)
        return tuple(v.detach() for v in (*out, loss, *torch.autograd.grad((out.logprob, out.entropy), (x, w), (up, up)),
                                          *torch.autograd.grad(loss, (x, w), up)))

    def inputs(size):
        return (torch.randn((2, 24, 128), generator=g, device=cuda).bfloat16(),
                torch.randint(0, 1000, (2, 24), generator=g, device=cuda),
                torch.randint(0, 1000, (2, 24, 6), generator=g, device=cuda),
                torch.randn((2, 24, 6), generator=g, device=cuda),
                size * torch.rand((2, 24), generator=g, device=cuda))

    graphed = GraphedStep(step, *inputs(1.0))
    for size in (100.0, 1e-3, 1.0):
        args = inputs(size)
        first = step(*args)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(*args)
        torch.cuda.current_stream().wait_stream(side)
        for a, b, c in zip(first, other, graphed(*args)):
            assert a.any() and torch.equal(a, b) and torch.equal(a, c)
