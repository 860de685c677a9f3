"""The token losses and AdamW as they are used together, and AdamW in the VGG16-BN step."""
import numpy as np
import pytest
import torch

from conftest import rel_l2

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def one(x, dtype=torch.float32):
    return torch.tensor([x], dtype=dtype, device="cuda")


class Head:
    """A linear policy head over fixed features: half working weights, float master weights."""

    def __init__(self, rows, features, classes, bits, seed=0):
        from renaissance_b200 import ops
        g = torch.Generator(device="cuda").manual_seed(seed)
        randn = lambda *s: torch.randn(s, generator=g, device="cuda")
        self.x = randn(rows, features).half()
        self.w = randn(classes, features) * features ** -0.5
        self.b = randn(classes) * 0.1
        self.w16 = self.w.half()
        self.gw, self.gb = torch.zeros_like(self.w), torch.zeros_like(self.b)
        z = lambda t, dtype=torch.float32: torch.zeros(t.shape, dtype=dtype, device="cuda")
        self.step = one(0, torch.int32)
        self.flag = one(0, torch.int32)
        self.scaling = one(1024.0)
        e4m3 = torch.float8_e4m3fn
        state = (lambda t: z(t)) if bits == 32 else (lambda t: torch.zeros(t.shape, dtype=torch.uint8, device="cuda").view(e4m3))
        self.m, self.v = [state(self.w), state(self.b)], [state(self.w), state(self.b)]
        blocks = lambda t: torch.zeros(-(-t.numel() // 128), device="cuda")
        more = {} if bits == 32 else dict(m_scales=[blocks(self.w), blocks(self.b)], v_scales=[blocks(self.w), blocks(self.b)])
        self.b16 = self.b.half()
        self.plan = ops.AdamWPlan([self.w, self.b], [self.gw, self.gb], self.m, self.v, copies=[self.w16, self.b16],
                                  weight_decay=[0.1, 0.0], **more)

    def logits(self):
        from renaissance_b200 import ops
        return ops.fc_amp_fwd(self.x, self.w16, self.b)

    def update(self, dlogits, lr=1e-2):
        from renaissance_b200 import ops
        ops.fc_amp_bwd(dlogits, self.w16, self.x, dw=self.gw, db=self.gb, want_dx=False)
        ops.check_nonfinite(self.gw.view(-1), self.flag)
        ops.check_nonfinite(self.gb, self.flag)
        ops.adamw_step(self.plan, self.step, lr, scaling=self.scaling, skip_flag=self.flag, seed=7)
        ops.grad_scaling(self.flag, self.scaling, clear_flag=True)


def rollout(head, classes, seed=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = head.x.shape[0]
    actions = torch.randint(0, classes, (rows,), generator=g, device="cuda", dtype=torch.int32)
    actions[::7] = -1
    adv = torch.randn(rows, generator=g, device="cuda")
    mask = (torch.rand(rows, generator=g, device="cuda") < 0.8).float()
    return actions, adv, mask / mask.sum()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("rows,features,classes", [(64, 128, 1000), (96, 64, 4096)])
def test_policy_step_against_autograd(rows, features, classes, bits):
    """log-probabilities of the acting and the reference policy -> loss and d logits -> FC backward -> AdamW, against the
    same step by autograd in double."""
    from renaissance_b200 import ops
    head = Head(rows, features, classes, bits)
    actions, adv, weights = rollout(head, classes)
    old = ops.token_logprobs(head.logits(), actions)["logp"]
    ref = old - 0.05
    w0, b0 = head.w.double(), head.b.double()
    out = ops.policy_loss_fused(head.logits(), actions, old, adv, head.scaling, ref_logp=ref, kl_coef=0.1, weights=weights)
    head.update(out["dlogits"])
    torch.cuda.synchronize()

    w = w0.half().double().requires_grad_()
    b = b0.clone().requires_grad_()
    z = head.x.double() @ w.t() + b
    rounded = z + (z.half().double() - z).detach()                       # the logits are stored in half
    ok = actions >= 0
    logp = torch.log_softmax(rounded, 1).gather(1, actions.long().clamp_min(0)[:, None])[:, 0]
    ratio = torch.exp(logp - old.double())
    gap = ref.double() - logp
    rowloss = -torch.minimum(ratio * adv.double(), ratio.clamp(0.8, 1.2) * adv.double()) + 0.1 * (torch.expm1(gap) - gap)
    loss = (rowloss * weights.double() * ok).sum()
    loss.backward()
    # logits: the GEMM's float sums, then half: one step of half where a sum sits next to a border (2^-10 of |z| < 8)
    assert abs(float(out["loss"]) - float(loss.detach())) < 2.0 ** -10 * 8
    # d logits carry half a step of half each (2^-11), the products are summed in float: the gradient's norm by 2^-9
    gw, gb = head.gw.double() / 1024.0, head.gb.double() / 1024.0
    assert rel_l2(gw.cpu().numpy(), w.grad.cpu().numpy()) < 2.0 ** -8
    assert rel_l2(gb.cpu().numpy(), b.grad.cpu().numpy()) < 2.0 ** -8
    # the first AdamW step from the gradients that the backward gave: m / sqrt(v) = sign(g), states from zero
    for got, start, g, decay in ((head.w, w0, gw, 0.1), (head.b, b0, gb, 0.0)):
        m, v = 0.1 * g, 0.001 * g * g
        want = start * (1 - 1e-2 * decay) - 1e-2 / 0.1 * m / ((v / 0.001).sqrt() + 1e-8)
        # 16 roundings of the change (1e-2 at most) and 4 of the weight; 1 - 0.999 in float: 2^-24 / 0.001 of v
        tol = 4 * U * start.abs() + (16 + 1000) * U * 1e-2
        assert ((got.double() - want).abs() <= tol).all()
    assert torch.equal(head.w16, head.w.half()) and int(head.step) == 1 and int(head.flag) == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_training_steps_equal_eager_ones(bits):
    """Log-probabilities, both losses and the update in one captured graph, replayed five times, against eager steps."""
    from renaissance_b200 import ops
    rows, classes = 64, 2048

    def step(head, data):
        actions, adv, weights, old, st = data
        z = head.logits()
        a = ops.policy_loss_fused(z, actions, old, adv, head.scaling, weights=weights)
        b = ops.preference_loss_fused(z, actions, st, None, head.scaling, beta=0.05)
        head.update(ops.add16(a["dlogits"], b["dlogits"]))
        return a["loss"], b["loss"], ops.token_logprobs(head.logits(), actions)["logp"]

    heads = [Head(rows, 128, classes, bits, seed=1) for _ in range(3)]
    actions, adv, weights = rollout(heads[0], classes)
    st = torch.tensor([0, 20, 30, 50, 60], dtype=torch.int32, device="cuda")
    data = (actions, adv, weights, ops.token_logprobs(heads[0].logits(), actions)["logp"], st)
    step(heads[2], data)                                                  # warm-up
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(heads[0], data)
    for i in range(5):
        graph.replay()
        eager = step(heads[1], data)
        torch.cuda.synchronize()
        for x, y in zip(captured, eager):
            assert torch.equal(x, y), i
    assert torch.equal(heads[0].w, heads[1].w) and int(heads[0].step) == 5
    bits_of = lambda t: t.view(torch.uint8) if t.element_size() == 1 else t
    for x, y in zip(heads[0].m + heads[0].v, heads[1].m + heads[1].v):
        assert torch.equal(bits_of(x), bits_of(y))


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
def test_vgg16bn_step_with_adamw(optimizer):
    """The trainer's gradients are SGD's; its update is AdamW of them.  A step with a non-finite gradient changes nothing
    but the loss scale."""
    from renaissance_b200.vgg16bn import Vgg16BnTrainer
    kw = dict(batch=4, image=32, classes=10, fc_width=256, dropout=0.0, lr=1e-3, weight_decay=0.1, seed=2)
    a = Vgg16BnTrainer(optimizer=optimizer, **kw)
    b = Vgg16BnTrainer(**kw)
    g = torch.Generator().manual_seed(0)
    images = torch.randn((4, 32, 32, 4), generator=g)
    images[..., 3] = 0
    for t in (a, b):
        t.images[0].copy_(images.half())
        t.labels[0].copy_(torch.tensor([1, 2, 3, 4], dtype=torch.int32))
    w0 = a.w32.clone()
    scaling = float(a.scaling)
    la, lb = float(a.step()), float(b.step())
    torch.cuda.synchronize()
    assert la == lb and torch.equal(a.g32, b.g32)
    grad = a.g32.double() / scaling
    decay = torch.zeros_like(w0)
    for s in a.slots:
        if len(s.shape) > 1:
            decay[s.offset:s.offset + s.stored] = 0.1
    want = w0.double() * (1 - 1e-3 * decay.double()) - 1e-3 * grad / (grad.abs() + 1e-8)
    # the update's roundings as in the operator's own test; 1 - beta2 in float: 2^-24 / 0.001 of v
    assert ((a.w32.double() - want).abs() <= 4 * U * w0.double().abs() + (16 + 1000) * U * 1e-3).all()
    for s in a.slots:                       # the copy, slot by slot (the gaps between slots are nobody's)
        assert torch.equal(a.w16[s.offset:s.offset + s.stored], a.w32[s.offset:s.offset + s.stored].half())
    assert int(a.adamw_steps) == 1
    before = [t.clone() for t in [a.w32] + a.adamw_states]
    a.scaling.fill_(float("inf"))
    a.step()
    torch.cuda.synchronize()
    assert int(a.adamw_steps) == 1
    for x, y in zip(before, [a.w32] + a.adamw_states):
        assert torch.equal(x, y)
    a.load_params(b.params())
    assert int(a.adamw_steps) == 0 and all(not t.any() for t in a.adamw_states)


def test_vgg16bn_refuses_other_optimizers():
    from renaissance_b200.vgg16bn import Vgg16BnTrainer
    with pytest.raises(ValueError):
        Vgg16BnTrainer(batch=4, image=32, classes=10, fc_width=256, optimizer="adam")
