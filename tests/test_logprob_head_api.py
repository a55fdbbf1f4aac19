"""Refusals of OutputHead.token_logprobs / distillation_loss and of the logit-row functions below them,
without a GPU: nothing may reach a kernel with fewer values than it has rows.  Tensors are fake ones on a
CUDA device (shapes and types, no data) or CPU tensors that no check here lets through to a launch."""
import pytest
import torch
from torch.autograd import forward_ad
from torch._subclasses import FakeTensorMode

from macrogpt_jax_b200 import _capi as C
from macrogpt_jax_b200 import ops

D, V = 16, 40


@pytest.fixture(params=["fused", "generic"])
def head(request):
    from macrogpt_jax_b200.einsum import Rngs
    from macrogpt_jax_b200.head import OutputHead
    h = OutputHead(D, V, rngs=Rngs(0))
    if request.param == "generic":
        h.norm.scale.data = h.norm.scale.data.float()
    assert h.fused() == (request.param == "fused")
    return h


@pytest.fixture
def launches(monkeypatch):
    """The logit-row entry points of the library replaced by a record of their rows."""
    calls = []
    for name in ("logprob_forward", "logprob_backward", "distill_forward", "distill_backward"):
        monkeypatch.setattr(C, name, lambda rows, *args, name=name: calls.append((name, rows.rows)))
    monkeypatch.setattr(ops, "_call_on", lambda t, kind, passes, fn, *args: fn(*args, None))
    return calls


def fake(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda")


@pytest.mark.parametrize("shape", [(2, 3, 2 * D), (2, 3, D // 2), (2, 3, D + 1), (2, D, 3), ()])
def test_head_refuses_activations_of_another_width(head, shape):
    lead = shape[:-1]
    with FakeTensorMode():
        x = fake(*shape)
        tok = fake(*lead, dtype=torch.int64)
        with pytest.raises(ValueError, match="token_logprobs: activations"):
            head.token_logprobs(x, tok)
        with pytest.raises(ValueError, match="distillation_loss: activations"):
            head.distillation_loss(x, fake(*lead, 4, dtype=torch.int64), fake(*lead, 4))


def test_head_loss_refuses_activations_of_another_width():
    """The loss of the same head flattens them in the same way."""
    from macrogpt_jax_b200.einsum import Rngs
    from macrogpt_jax_b200.head import OutputHead
    h = OutputHead(D, V, rngs=Rngs(0))
    with FakeTensorMode():
        for width in (2 * D, D // 2):
            with pytest.raises(ValueError, match="token_loss: activations"):
                h.token_loss(fake(2, 3, width), fake(2, 3, dtype=torch.int64))


@pytest.mark.parametrize("n", [6, 13])
def test_loss_functions_refuse_other_numbers_of_labels(n):
    with FakeTensorMode():
        x, row = fake(12, V), fake(12, dtype=torch.float32)
        stats = fake(12, 1, 2, dtype=torch.float32)
        good, lab, mk = fake(12, dtype=torch.int32), fake(n, dtype=torch.int32), fake(n, dtype=torch.uint8)
        for labels, mask in ((lab, None), (good, mk), (fake(12, dtype=torch.int64), None)):
            for call in (lambda: ops.xent_rows(x, labels, mask), lambda: ops.xent_combine(stats, x, V, labels, mask),
                         lambda: ops.xent_grad(x, labels, mask, row, row, row, 0.0, C.E5M2)):
                with pytest.raises(ValueError, match="cross-entropy"):
                    call()


def split_head(monkeypatch, rank=1, ranks=4):
    """A head whose lm_head weight was split by Einsum.reshard, without a process group."""
    import torch.distributed as dist
    from macrogpt_jax_b200 import tp
    from macrogpt_jax_b200.einsum import Rngs
    from macrogpt_jax_b200.head import OutputHead
    h = OutputHead(D, V, rngs=Rngs(0))
    monkeypatch.setattr(tp, "tensor_group", lambda mesh: "group")
    monkeypatch.setattr(dist, "get_world_size", lambda group: ranks)
    monkeypatch.setattr(dist, "get_rank", lambda group: rank)
    h.lm_head.reshard(object())
    assert h.lm_head.w.shape == (D, V // ranks) and not h.fused()
    return h


def test_split_head_is_refused(monkeypatch):
    """This rank's columns alone would give the entropy, alternatives and loss of a part of the vocabulary."""
    h = split_head(monkeypatch)
    with FakeTensorMode():
        x, tok = fake(2, 3, D), fake(2, 3, dtype=torch.int64)
        with pytest.raises(NotImplementedError, match="token_logprobs: the lm_head holds part 1 of 4"):
            h.token_logprobs(x, tok)
        with pytest.raises(NotImplementedError, match="distillation_loss: the lm_head holds part 1 of 4"):
            h.distillation_loss(x, fake(2, 3, 4, dtype=torch.int64), fake(2, 3, 4))


def test_loss_of_a_split_head_is_refused(monkeypatch):
    """The same for the next-token loss, whichever way the head is given."""
    from macrogpt_jax_b200.next_token_loss import chunked_softmax_cross_entropy
    h = split_head(monkeypatch)
    with FakeTensorMode():
        x, tok = fake(2, 3, D), fake(2, 3, dtype=torch.int64)
        for projection in (h, h.get_logits, h.forward):
            with pytest.raises(NotImplementedError, match="cross_entropy: the lm_head holds part 1 of 4"):
                chunked_softmax_cross_entropy(tok, x, projection)


@pytest.mark.parametrize("lead", [(2, 3), (5,), (), (0,)])
@pytest.mark.parametrize("k", [0, 1, 4])
def test_head_takes_any_number_of_entries(monkeypatch, lead, k):
    """No entries at all included, as topk_distillation_loss takes them."""
    from macrogpt_jax_b200 import head as hd
    from macrogpt_jax_b200.einsum import Rngs
    seen = []
    monkeypatch.setattr(hd.OutputHead, "_rows",
                        lambda self, x, op, who: seen.append(op) or (x.new_empty(x.shape[:-1].numel()),))
    h = hd.OutputHead(D, V, rngs=Rngs(0))
    with FakeTensorMode():
        loss = h.distillation_loss(fake(*lead, D), fake(*lead, k, dtype=torch.int64), fake(*lead, k))
    rows = torch.Size(lead).numel()
    assert loss.shape == lead and seen[0].ids.shape == (rows, k) and seen[0].teacher.shape == (rows, k)


def on(device, h):
    """The head with fake parameters on the device."""
    for m in (h.norm, h.lm_head):
        for name, p in list(m.named_parameters()):
            setattr(m, name, torch.nn.Parameter(torch.empty(p.shape, dtype=p.dtype, device=device)))
    return h


def test_head_runs_on_its_device(monkeypatch):
    """Activations on another device than the current one: the whole node runs with that device current;
    activations on another device than the head: refused."""
    import contextlib
    from macrogpt_jax_b200.einsum import Rngs
    from macrogpt_jax_b200.head import OutputHead
    current, seen = [0], []

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], torch.device(d).index
        try:
            yield
        finally:
            current[0] = before

    def forward(x2d, scale, centered, eps, w, cap):
        seen.append(current[0])
        raise StopIteration

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(ops, "head_rows_forward", forward)
    with FakeTensorMode():
        h = OutputHead(D, V, rngs=Rngs(0))
        x = torch.empty((2, D), dtype=torch.bfloat16, device="cuda:1")
        tok = torch.empty(2, dtype=torch.int64, device="cuda:1")
        ids, t = torch.empty((2, 3), dtype=torch.int64, device="cuda:1"), torch.empty((2, 3), device="cuda:1")
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                on("cuda:1", h)
                for call in (lambda: h.token_logprobs(x, tok), lambda: h.distillation_loss(x, ids, t)):
                    with pytest.raises(StopIteration):
                        call()
                    assert seen.pop() == 1 and current == [0]
                on("cuda:0", h)
                for call in (lambda: h.token_logprobs(x, tok), lambda: h.distillation_loss(x, ids, t)):
                    with pytest.raises(ValueError, match="the head on cuda:0"):
                        call()
    assert not seen


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(grad):
    """A tangent without requires_grad would be dropped: a derivative of zero without a word."""
    from macrogpt_jax_b200.distill import topk_distillation_loss
    from macrogpt_jax_b200.einsum import Rngs
    from macrogpt_jax_b200.head import OutputHead
    from macrogpt_jax_b200.logprobs import token_logprobs
    h = OutputHead(D, V, rngs=Rngs(0)).requires_grad_(False)
    with FakeTensorMode(allow_non_fake_inputs=True), forward_ad.dual_level(), torch.set_grad_enabled(grad):
        def dual(*shape, dtype=torch.float32):
            return forward_ad.make_dual(fake(*shape, dtype=dtype), fake(*shape, dtype=dtype))
        tok, ids, t = fake(2, dtype=torch.int64), fake(2, 3, dtype=torch.int64), fake(2, 3)
        for call in (lambda: token_logprobs(dual(2, V), tok),
                     lambda: topk_distillation_loss(dual(2, V), ids, t),
                     lambda: topk_distillation_loss(fake(2, V), ids, dual(2, 3)),
                     lambda: h.token_logprobs(dual(2, D, dtype=torch.bfloat16), tok),
                     lambda: h.token_logprobs(dual(2, D), tok),
                     lambda: h.distillation_loss(dual(2, D), ids, t),
                     lambda: h.distillation_loss(fake(2, D), ids, dual(2, 3))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


ROWS = 12


def args(n=ROWS, k=3):
    """(logits of ROWS rows, tokens, mask, ids, teacher, stats, upstream, dtop) for n rows."""
    return (torch.zeros(ROWS, V), torch.zeros(n, dtype=torch.int64), torch.ones(n, dtype=torch.bool),
            torch.zeros(n, k, dtype=torch.int64), torch.zeros(n, k), torch.zeros(n, 4), torch.zeros(n),
            torch.zeros(n, k))


def test_functions_take_matching_rows(launches):
    x, tok, mask, ids, teacher, stats, up, dtop = args()
    ops.token_logprobs_forward(x, tok, mask, 3, 1.0, True, True)
    ops.token_logprobs_backward(x, stats, tok, mask, 1.0, up, up, dtop, ids)
    ops.distill_forward(x, ids, teacher, mask, 1.0, True)
    ops.distill_backward(x, stats, ids, teacher, mask, 1.0, up.sum().expand(ROWS))
    assert launches == [(n, ROWS) for n in ("logprob_forward", "logprob_backward", "distill_forward",
                                            "distill_backward")]


@pytest.mark.parametrize("n", [6, 11, 13, 24])
@pytest.mark.parametrize("which", range(12))
def test_functions_refuse_other_numbers_of_rows(launches, n, which):
    x, tok, mask, ids, teacher, stats, up, dtop = args()
    _, tok2, mask2, ids2, teacher2, stats2, up2, dtop2 = args(n)
    bad = [lambda: ops.token_logprobs_forward(x, tok2, None, 0, 1.0, True, True),
           lambda: ops.token_logprobs_forward(x, tok, mask2, 0, 1.0, True, True),
           lambda: ops.token_logprobs_backward(x, stats, tok2, None, 1.0, up, None, None, None),
           lambda: ops.token_logprobs_backward(x, stats, tok, mask2, 1.0, up, None, None, None),
           lambda: ops.token_logprobs_backward(x, stats2, tok, None, 1.0, up, None, None, None),
           lambda: ops.token_logprobs_backward(x, stats, tok, None, 1.0, up2, None, None, None),
           lambda: ops.token_logprobs_backward(x, stats, tok, None, 1.0, None, up2, None, None),
           lambda: ops.token_logprobs_backward(x, stats, tok, None, 1.0, None, None, dtop2, ids),
           lambda: ops.distill_forward(x, ids2, teacher2, None, 1.0, True),
           lambda: ops.distill_forward(x, ids, teacher, mask2, 1.0, True),
           lambda: ops.distill_backward(x, stats, ids, teacher2, None, 1.0, up),
           lambda: ops.distill_backward(x, stats, ids, teacher, None, 1.0, up2)][which]
    with pytest.raises(ValueError, match="logit rows"):
        bad()
    assert launches == []


@pytest.mark.parametrize("call", [
    lambda x, tok, mask, ids, t: ops.token_logprobs_forward(x, tok.to(torch.int16), None, 0, 1.0, True, True),
    lambda x, tok, mask, ids, t: ops.token_logprobs_forward(x, tok, mask.int(), 0, 1.0, True, True),
    lambda x, tok, mask, ids, t: ops.distill_forward(x, ids.to(torch.int16), t, None, 1.0, True),
    lambda x, tok, mask, ids, t: ops.distill_forward(x, ids, t, mask.long(), 1.0, True),
])
def test_functions_refuse_other_types(launches, call):
    """Narrower ids would be read past their end, wider masks in pieces."""
    with pytest.raises(TypeError, match="logit rows"):
        call(*args()[:5])
    assert launches == []


def test_exact_amax_flag():
    """UFP8_AMAX_EXACT goes with the two fp8 formats, and with nothing else."""
    import ctypes
    import re
    from pathlib import Path
    header = (Path(__file__).resolve().parents[1] / "include" / "ufp8.h").read_text()
    assert int(re.search(r"#define UFP8_AMAX_EXACT (\d+)", header)[1]) == C.AMAX_EXACT
    p = 1 << 20  # stands for an aligned device address; no call here reads it
    lib = C.load()

    def call(fmt, dtype=C.OUT_BF16, cap=0.0, amax=p):
        r = C.LogitRows(p, dtype, 1.0, 4, 100, 4, 0, 100, None)
        a = lib.ufp8_logprob_backward(ctypes.byref(r), p, p, 8, p, 1, None, 0, None, None, 0, cap, fmt, p, 400, 100,
                                      amax, p, None), lib.ufp8_last_error().decode()
        b = lib.ufp8_distill_backward(ctypes.byref(r), p, p, 8, p, C.OUT_F32, 4, p, 1, cap, fmt, p, 400, 100, amax, p,
                                      None), lib.ufp8_last_error().decode()
        return a, b

    for rc, msg in call(C.BF16 | C.AMAX_EXACT) + call(5 | C.AMAX_EXACT) + call(2 * C.AMAX_EXACT):
        assert rc == C.ERR_INVALID and "fmt" in msg
    for fmt in (C.E4M3, C.E5M2):
        for rc, msg in call(fmt | C.AMAX_EXACT, dtype=C.OUT_F32):
            assert rc == C.ERR_UNSUPPORTED and "bf16" in msg
        for rc, msg in call(fmt | C.AMAX_EXACT, amax=None):
            assert rc == C.ERR_INVALID and "null amax" in msg


@pytest.mark.parametrize("fmt", [C.E4M3, C.E5M2])
def test_head_backward_asks_for_the_scale_that_its_format_needs(monkeypatch, fmt):
    """e5m2 takes the bound of the rows' results; e4m3, whose range it would use up, the largest value."""
    asked = []

    def grad(logits, head):
        asked.append(head)
        return ops.Fp8Tensor(torch.empty(3, 48, dtype=ops.FP8_DTYPE[fmt]), None, None)

    monkeypatch.setattr(ops, "gemm", lambda *a, **k: None)
    monkeypatch.setattr(ops, "operand", lambda *a: None)
    q = ops.Fp8Tensor(torch.empty(3, D), None, None)
    ops.head_rows_backward(grad, torch.empty(3, 48), (q, None, q), V, 15.0, True, fmt)
    assert asked == [(15.0, C.E5M2 if fmt == C.E5M2 else C.E4M3 | C.AMAX_EXACT, 48)]
