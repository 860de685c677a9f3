"""GPU parity of the AdamW step over many tensors with its definition: in 64 bits for float states, and for 8-bit
states also code by code against the same float operations done by numpy.

u = 2^-24.  A state is a sum of two products: |m| terms carry 4 roundings (unscaled gradient, constant, product, sum), v
terms 5.  The weight's change carries those of m (4) and half of v's (3), square root, two products, a sum, a division
and the bias corrections: counted as 16; the weight itself two products and a sum."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SIZES = [1, 2, 3, 4, 127, 128, 129, 255, 256, 257, 384, 1000, 4095, 4096, 4097, 8192 + 300, 70001]
LR, B1, B2, EPS = 3e-3, 0.9, 0.999, 1e-8


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def one(x, dtype=torch.float32):
    return torch.tensor([x], dtype=dtype, device="cuda")


def place(values, skip):
    """The same values `skip` elements behind an aligned address, with sentinels around them."""
    n = values.numel()
    flat = torch.zeros(n + skip + 16, dtype=values.dtype, device="cuda")
    if values.element_size() == 1:
        flat.view(torch.uint8).fill_(0x55)
        flat.view(torch.uint8)[skip:skip + n] = values.view(torch.uint8)
    else:
        flat.fill_(-77.0)
        flat[skip:skip + n] = values
    return flat, flat[skip:skip + n]


def untouched(flat, n, skip):
    want = 0x55 if flat.element_size() == 1 else -77.0
    f = flat.view(torch.uint8) if flat.element_size() == 1 else flat
    return bool((f[:skip] == want).all() and (f[skip + n:] == want).all())


def tensors(sizes, grad, copy, seed=0, skips=None, eight=False, started=True):
    g = gen(seed)
    skips = skips or [0] * len(sizes)
    t = dict(w=[], g=[], m=[], v=[], ms=[], vs=[], c=[])
    flats = []
    for n, skip in zip(sizes, skips):
        def put(key, x):
            f, view = place(x, skip)
            flats.append((f, n if key not in ("ms", "vs") else x.numel(), skip))
            t[key].append(view)
        randn = lambda: torch.randn(n, generator=g, device="cuda")
        scale = torch.exp(2 * randn())
        put("w", randn() * 0.1)
        put("g", (randn() * scale).to(grad))
        m, v = randn() * scale * 0.1 * started, (scale * randn()) ** 2 * 0.01 * started
        if eight:
            k = -(-n // 128)
            codes = lambda lo: torch.randint(lo, 0x7f, (n,), generator=g, device="cuda", dtype=torch.uint8)
            sign = torch.randint(0, 2, (n,), generator=g, device="cuda", dtype=torch.uint8) * 128
            put("m", ((codes(0) | sign) * int(started)).view(torch.float8_e4m3fn))
            put("v", (codes(0) * int(started)).view(torch.float8_e4m3fn))
            put("ms", torch.rand(k, generator=g, device="cuda") * 1e-3 * started)
            put("vs", torch.rand(k, generator=g, device="cuda") * 1e-4 * started)
        else:
            put("m", m)
            put("v", v)
        if copy is not None:
            put("c", torch.zeros(n, dtype=copy, device="cuda"))
    return t, flats


def plan_of(t, decay, eight):
    from renaissance_b200 import ops
    return ops.AdamWPlan(t["w"], t["g"], t["m"], t["v"], t["ms"] if eight else None, t["vs"] if eight else None,
                         t["c"] or None, decay)


def clone(t):
    return {k: [x.clone() for x in v] for k, v in t.items()}


def check32(got, old, decay, step, lr=LR, scaling=1.0, b1=B1, b2=B2, eps=EPS):
    t = step + 1
    for i, w in enumerate(old["w"]):
        g = old["g"][i].double() / scaling
        m0, v0 = old["m"][i].double(), old["v"][i].double()
        m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
        upd = lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps)
        want = w.double() * (1 - lr * decay[i]) - upd
        m_tol = 4 * U * (b1 * m0.abs() + (1 - b1) * g.abs())
        size = lr / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + eps)
        assert ((got["m"][i].double() - m).abs() <= m_tol + 1e-44).all()
        assert ((got["v"][i].double() - v).abs() <= 5 * U * v + 1e-44).all()
        assert ((got["w"][i].double() - want).abs() <= 4 * U * w.double().abs() + 16 * U * upd.abs() + size * m_tol + 1e-44).all(), i
        if got["c"]:
            assert torch.equal(got["c"][i], got["w"][i].to(got["c"][i].dtype))


@pytest.mark.parametrize("copy", [None, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("grad", [torch.float32, torch.float16, torch.bfloat16])
def test_float_states(grad, copy):
    from renaissance_b200 import ops
    for skips in (None, [i % 9 for i in range(len(SIZES))]):
        t, flats = tensors(SIZES, grad, copy, seed=1, skips=skips)
        decay = [0.1 * (i % 2) for i in range(len(SIZES))]
        old = clone(t)
        step = one(6, torch.int32)
        ops.adamw_step(plan_of(t, decay, False), step, LR, scaling=one(128.0))
        check32(t, old, decay, 6, scaling=128.0)
        assert int(step) == 7
        assert all(untouched(*f) for f in flats)


def test_first_and_late_steps_and_constants():
    from renaissance_b200 import ops
    for step, lr, b1, b2, eps in ((0, 1e-3, 0.9, 0.999, 1e-8), (0, 0.5, 0.0, 0.0, 1e-6), (1, 1e-2, 0.95, 0.99, 1e-15),
                                  (2_000_000, 1e-4, 0.9, 0.9999, 1e-8), (10, 0.0, 0.9, 0.999, 1e-8)):
        t, _ = tensors([1000, 77], torch.float32, None, seed=2, started=step > 0)
        old = clone(t)
        n = one(step, torch.int32)
        ops.adamw_step(plan_of(t, 0.01, False), n, lr, b1, b2, eps)
        check32(t, old, [0.01, 0.01], step, lr=lr, b1=b1, b2=b2, eps=eps)
        assert int(n) == step + 1


def test_empty_tensors_among_others():
    from renaissance_b200 import ops
    t, _ = tensors([0, 5, 0, 130], torch.float32, None, seed=3)
    old = clone(t)
    step = one(0, torch.int32)
    ops.adamw_step(plan_of(t, 0.0, False), step, LR)
    check32(t, old, [0.0] * 4, 0)
    t, _ = tensors([0], torch.float32, None)
    ops.adamw_step(plan_of(t, 0.0, False), step, LR)
    assert int(step) == 2


@pytest.mark.parametrize("eight", [False, True])
def test_skip_flag_stops_everything(eight):
    from renaissance_b200 import ops
    t, _ = tensors([300, 5000], torch.float32, torch.float16, seed=4, eight=eight)
    t["g"][0][7] = math.inf
    old = clone(t)
    step, flag = one(3, torch.int32), one(1, torch.int32)
    plan = plan_of(t, 0.1, eight)
    ops.adamw_step(plan, step, LR, skip_flag=flag)
    assert int(step) == 3
    bits = lambda x: x.view(torch.uint8) if x.element_size() == 1 else x
    for k in old:
        for a, b in zip(old[k], t[k]):
            assert torch.equal(bits(a), bits(b))
    flag.zero_()
    t["g"][0][7] = 1.0
    ops.adamw_step(plan, step, LR, skip_flag=flag)
    assert int(step) == 4 and not torch.equal(old["w"][1], t["w"][1])


def test_captured_steps_follow_step_and_rate():
    from renaissance_b200 import ops
    a, _ = tensors([300, 5000, 17], torch.bfloat16, torch.bfloat16, seed=5, started=False)
    b = clone(a)
    pa, pb = plan_of(a, 0.1, False), plan_of(b, 0.1, False)
    sa, sb, lr = one(0, torch.int32), one(0, torch.int32), one(LR)
    g = torch.cuda.CUDAGraph()
    warm = clone(a)
    ops.adamw_step(plan_of(warm, 0.1, False), one(0, torch.int32), lr)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        ops.adamw_step(pa, sa, lr)
    for i in range(5):
        rate = float(torch.tensor(LR / (i + 1), dtype=torch.float32))
        lr.fill_(rate)
        g.replay()
        ops.adamw_step(pb, sb, rate)
    torch.cuda.synchronize()
    assert int(sa) == int(sb) == 5
    for k in ("w", "m", "v", "c"):
        for x, y in zip(a[k], b[k]):
            assert torch.equal(x, y)


@pytest.mark.parametrize("eight", [False, True])
def test_plans_on_two_streams_and_many_tensors(eight):
    """Two plans of 700 tensors each step at once on two streams; the results are those of one after the other."""
    from renaissance_b200 import ops
    sizes = [1 + (i * 37) % 900 for i in range(697)] + [0, 300_000, 5]
    sets = [tensors(sizes, torch.float16, torch.bfloat16, seed=s, eight=eight, started=False)[0] for s in (1, 2)]
    want = [clone(t) for t in sets]
    for t in want:
        n = one(0, torch.int32)
        p = plan_of(t, 0.1, eight)
        for _ in range(3):
            ops.adamw_step(p, n, LR, seed=5)
    plans = [plan_of(t, 0.1, eight) for t in sets]
    steps = [one(0, torch.int32) for _ in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(3):
        for p, n, s in zip(plans, steps, streams):
            ops.adamw_step(p, n, LR, seed=5, stream=s)
    torch.cuda.synchronize()
    bits = lambda x: x.view(torch.uint8) if x.element_size() == 1 else x
    for got, ref, n in zip(sets, want, steps):
        assert int(n) == 3
        for k in ref:
            for a, b in zip(got[k], ref[k]):
                assert torch.equal(bits(a), bits(b)), k


# ------------------------------------------------------------------------------------------------ 8-bit states

def philox(counter, key):
    c = [x.astype(np.uint64) for x in counter]
    k = [np.uint64(key & 0xFFFFFFFF), np.uint64(key >> 32)]
    low, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> sh) ^ c[1] ^ k[0], p1 & low, (p0 >> sh) ^ c[3] ^ k[1], p0 & low]
        k = [(k[0] + np.uint64(0x9E3779B9)) & low, (k[1] + np.uint64(0xBB67AE85)) & low]
    return c


def halves(n, tensor, step, seed):
    """The 16 random bits of each element."""
    i = np.arange(n)
    block, lane, j = i // 128, i % 128 // 4, i % 4
    group = (block // 2) * 32 + lane
    words = philox([group & 0xFFFFFFFF, np.full(n, tensor), np.full(n, step), group >> 32], seed)
    word = np.stack(words)[j, i]
    return np.where(block % 2, word >> np.uint64(16), word & np.uint64(0xFFFF)).astype(np.uint32)


TABLE = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()


def codes(x):
    return x.view(torch.uint8).cpu().numpy()


def pack(x, random=None):
    """numpy's float32 version of the storage: (codes, scales)."""
    n = len(x)
    k = -(-n // 128)
    y = np.zeros(k * 128, np.float32)
    y[:n] = x
    y = y.reshape(k, 128)
    top = np.abs(y).max(1)
    small = top < np.float32(2.0 ** -116)
    safe = np.where(small, np.float32(1), top)
    up = np.where(small, np.float32(0), np.float32(1) / safe * np.float32(448)).astype(np.float32)
    scale = np.where(small, np.float32(0), top * np.float32(1 / np.float32(448))).astype(np.float32)
    y = (y * up[:, None]).reshape(-1)[:n]
    if random is None:
        q = torch.from_numpy(np.clip(y, -448, 448)).to(torch.float8_e4m3fn)
        return q.view(torch.uint8).numpy(), scale
    y = np.minimum(y, np.float32(448))
    normal = y >= np.float32(2.0 ** -6)
    bits = np.where(normal, y, y + np.float32(2.0 ** -6)).astype(np.float32).view(np.uint32)
    c = ((bits + (random << np.uint32(4))) >> np.uint32(20)) - np.where(normal, 960, 968).astype(np.uint32)
    return np.where((c == 0) & (y > 0), 1, c).astype(np.uint8), scale


def step8(old, i, step, seed, scaling, decay, lr=LR):
    f = np.float32
    n = old["w"][i].numel()
    block = np.arange(n) // 128
    g = old["g"][i].float().cpu().numpy() * (f(1) / f(scaling))
    m = TABLE[codes(old["m"][i])] * old["ms"][i].cpu().numpy()[block]
    v = TABLE[codes(old["v"][i])] * old["vs"][i].cpu().numpy()[block]
    m = m * f(B1) + g * f(1 - B1)
    v = v * f(B2) + (g * g) * f(1 - B2)
    t = step + 1
    w = old["w"][i].cpu().numpy().astype(np.float64) * (1 - lr * decay)
    upd = lr / (1 - B1 ** t) * m.astype(np.float64) / (np.sqrt(v.astype(np.float64) / (1 - B2 ** t)) + EPS)
    return w - upd, np.abs(upd), m, v, pack(m), pack(v, halves(n, i, step, seed))


@pytest.mark.parametrize("copy", [None, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("grad", [torch.float32, torch.float16, torch.bfloat16])
def test_8bit_states_code_by_code(grad, copy):
    from renaissance_b200 import ops
    for seed, skips, started in ((0, None, True), ((7 << 32) + 11, [i % 5 for i in range(len(SIZES))], True), (5, None, False)):
        t, flats = tensors(SIZES, grad, copy, seed=6, skips=skips, eight=True, started=started)
        decay = [0.1 * (i % 2) for i in range(len(SIZES))]
        old = clone(t)
        step = one(41 * started, torch.int32)
        s0 = int(step)
        ops.adamw_step(plan_of(t, decay, True), step, LR, scaling=one(4.0), seed=seed)
        assert int(step) == s0 + 1
        for i, n in enumerate(SIZES):
            w, upd, m, v, (mc, ms), (vc, vs) = step8(old, i, s0, seed, 4.0, decay[i])
            assert np.array_equal(codes(t["m"][i]), mc) and np.array_equal(t["ms"][i].cpu().numpy(), ms), n
            assert np.array_equal(codes(t["v"][i]), vc) and np.array_equal(t["vs"][i].cpu().numpy(), vs), n
            got = t["w"][i].cpu().numpy().astype(np.float64)
            assert (np.abs(got - w) <= 4 * U * np.abs(old["w"][i].cpu().numpy()) + 16 * U * upd + 1e-44).all(), n
            if copy is not None:
                assert torch.equal(t["c"][i], t["w"][i].to(copy))
        assert all(untouched(*f) for f in flats)


def test_8bit_states_of_extreme_blocks():
    """Blocks of zeros, of numbers too small to scale, of one large and many tiny ones, with an infinity."""
    from renaissance_b200 import ops
    n = 128 * 6
    t, _ = tensors([n], torch.float32, None, seed=7, eight=True, started=False)
    g = t["g"][0].view(6, 128)
    g[0] = 0
    g[1] = 1e-19                            # v = 1e-41: a denormal block
    g[2] = 1e-9
    g[2, 5] = 1e9
    g[3] = 1e17
    g[4, 100] = math.inf
    old = clone(t)
    ops.adamw_step(plan_of(t, 0.0, True), one(0, torch.int32), LR, seed=3)
    m, v = t["m"][0].float().view(6, 128), t["v"][0].float().view(6, 128)
    ms, vs = t["ms"][0], t["vs"][0]
    assert not m[0].any() and not v[0].any() and float(ms[0]) == 0 and float(vs[0]) == 0
    assert float(vs[1]) == 0 and not v[1].any()
    assert v[2, 5] == 448 and (v[2, :5] == 2.0 ** -9).all()          # tiny, but never zero
    assert v[3].isfinite().all() and abs(float(v[3, 0] * vs[3]) / (1e34 * (1 - B2)) - 1) < 2.0 ** -3
    assert (m[4] * ms[4]).isnan().all() and (v[4] * vs[4]).isnan().all()
    assert (m[5] * ms[5]).isfinite().all() and t["w"][0].view(6, 128)[[0, 1, 2, 3, 5]].isfinite().all()
    assert torch.equal(t["w"][0].view(6, 128)[0], old["w"][0].view(6, 128)[0])


def test_stochastic_rounding_keeps_the_mean():
    """Many elements with the same v: the mean of what is stored is v within six standard deviations, other seeds and
    steps draw other bits, the same ones the same."""
    from renaissance_b200 import ops
    n = 1 << 20

    def stored(seed, step):
        z = lambda dtype: torch.zeros(n, dtype=dtype, device="cuda")
        g = torch.full((n,), 0.61, device="cuda")
        g[::128] = 1.0                      # sets each block's scale
        t = dict(w=[z(torch.float32)], g=[g], m=[z(torch.uint8).view(torch.float8_e4m3fn)],
                 v=[z(torch.uint8).view(torch.float8_e4m3fn)], ms=[torch.zeros(n // 128, device="cuda")],
                 vs=[torch.zeros(n // 128, device="cuda")], c=[])
        ops.adamw_step(plan_of(t, 0.0, True), one(step, torch.int32), LR, seed=seed)
        return t["v"][0].float().view(-1, 128)[:, 1:].double(), float(t["vs"][0][0])

    v, scale = stored(1, 0)
    y = 0.61 ** 2 * 448                     # between the codes 160 and 176
    assert set(v.unique().tolist()) == {160.0, 176.0}
    share = (y - 160) / 16
    sd = math.sqrt(share * (1 - share) / v.numel())
    assert abs(float((v == 176).double().mean()) - share) < 6 * sd + 2.0 ** -16
    assert torch.equal(stored(1, 0)[0], v)
    for other in (stored(2, 0)[0], stored(1, 1)[0], stored(1 << 33, 0)[0]):
        agree = float((other == v).double().mean())
        assert abs(agree - (share ** 2 + (1 - share) ** 2)) < 0.01


def test_plan_refuses_on_device():
    from renaissance_b200 import _lib, ops
    f = lambda n=8, dtype=torch.float32: torch.zeros(n, dtype=dtype, device="cuda")
    w = f()
    with pytest.raises(_lib.Trb200Error):
        ops.AdamWPlan([w, w], [f(), f()], [f(), f()], [f(), f()])
    with pytest.raises(_lib.Trb200Error):
        ops.AdamWPlan([w], [f()], [w], [f()])
    with pytest.raises(TypeError):
        ops.AdamWPlan([f(8, torch.float16)], [f()], [f()], [f()])
    with pytest.raises(TypeError):
        ops.AdamWPlan([w, f()], [f(), f(8, torch.float16)], [f(), f()], [f(), f()])
    with pytest.raises(TypeError):
        ops.AdamWPlan([w], [f()], [f()], [f()], copies=[f()])
    with pytest.raises(ValueError):
        ops.AdamWPlan([w], [f(7)], [f()], [f()])
    with pytest.raises(ValueError):
        ops.AdamWPlan([w], [f()], [f(8, torch.float8_e4m3fn)], [f(8, torch.float8_e4m3fn)])
    with pytest.raises(ValueError):
        ops.AdamWPlan([f(200)], [f(200)], [f(200, torch.float8_e4m3fn)], [f(200, torch.float8_e4m3fn)], [f(1)], [f(1)])
    with pytest.raises(ValueError):
        ops.AdamWPlan([f(64).view(8, 8).t()], [f(64)], [f(64)], [f(64)])
    plan = ops.AdamWPlan([w], [f()], [f()], [f()])
    step = one(0, torch.int32)
    with pytest.raises(TypeError):
        ops.adamw_step(plan, one(0.0), LR)
    with pytest.raises(TypeError):
        ops.adamw_step(plan, step, one(1, torch.int32))
    with pytest.raises(_lib.Trb200Error):
        ops.adamw_step(plan, step, LR, beta1=1.0)
    with pytest.raises(_lib.Trb200Error):
        ops.adamw_step(plan, step, LR, eps=0.0)


# ------------------------------------------------------------------------------------------------ tiny second moments

def least_eps(beta2, eight):
    return 2.0 ** (-53 if eight else -55) / math.sqrt(1 - beta2)


def zero_states(g, eight, w=0.0):
    n = g.numel()
    state = lambda: torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) if eight else torch.zeros(n, device="cuda")
    t = dict(w=[torch.full((n,), w, device="cuda")], g=[g], m=[state()], v=[state()], c=[])
    if eight:
        t["ms"], t["vs"] = ([torch.zeros(-(-n // 128), device="cuda")] for _ in range(2))
    return t


@pytest.mark.parametrize("beta2", [0.99, 0.999, 0.9999])
@pytest.mark.parametrize("eight", [False, True])
def test_first_step_with_tiny_gradients_and_eps(eight, beta2):
    """v of the first step is subnormal from |g| = 3e-18 down (beta2 = 0.999): the change is that of the 64-bit formula for
    every decade of eps that is accepted.  Off by the 16 + 4 roundings of the change, and by sqrt(2^-149 / (1 - beta2))
    in the denominator."""
    from renaissance_b200 import ops
    g = torch.tensor([s * x for x in (1e-12, 1e-15, 1e-16, 1e-17, 3e-18, 1e-18, 1e-19, 1e-20, 1e-21, 1e-22, 1e-25) for s in (1, -1)],
                     device="cuda").repeat(13)
    least = least_eps(beta2, eight)
    for eps in [least * 1.01] + [10.0 ** -k for k in range(4, 16) if 10.0 ** -k >= least]:
        t = zero_states(g, eight)
        eps = float(torch.tensor(eps, dtype=torch.float32))
        ops.adamw_step(plan_of(t, 0.0, eight), one(0, torch.int32), 1.0, 0.9, beta2, eps)
        want = -g.double() / (g.double().abs() + eps)
        off = (t["w"][0].double() - want).abs()
        rel = 20 * U + U / (1 - beta2) + 2.0 ** -74.5 / math.sqrt(1 - beta2) / eps      # 1 - beta2 is a float, too
        assert (off <= rel * want.abs() + 1e-44).all(), (eps, float((off / want.abs()).max()))


@pytest.mark.parametrize("x", [3e-17, 1e-18, 1e-19, 1e-20, 1e-21, 1e-23])
def test_many_steps_with_tiny_gradients(x):
    """Constant gradients at the smallest eps: every step changes the weight by lr g / (|g| + eps), whatever v loses."""
    from renaissance_b200 import ops
    beta2, steps = 0.999, 300
    eps = float(torch.tensor(least_eps(beta2, False) * 1.01, dtype=torch.float32))
    g = torch.full((260,), x, device="cuda")
    g[1::2] *= -1
    t = zero_states(g, False)
    plan, n = plan_of(t, 0.0, False), one(0, torch.int32)
    for _ in range(steps):
        ops.adamw_step(plan, n, 1.0, 0.9, beta2, eps)
    want = -steps * g.double() / (g.double().abs() + eps)
    # a step: 16 roundings, 4 / (1 - 0.9) that m gathers, beta2's and 1 - beta2's own, 5 / (1 - beta2) that v gathers, half of
    # that in its root, what v loses where it is subnormal; and a rounding of the weight, which is at most `want`
    rel = (56 + steps) * U + (0.5 + 2.5) * U / (1 - beta2) + 2.0 ** -74.5 / math.sqrt(1 - beta2) / eps
    off = (t["w"][0].double() - want).abs()
    assert (off <= rel * want.abs()).all(), float((off / want.abs()).max())


@pytest.mark.parametrize("x", [1e-12, 1e-16, 1e-17, 1e-18, 1e-20])
def test_many_8bit_steps_with_tiny_gradients(x):
    """8-bit v below 2^-116 is stored as zeros, which takes at most 2^-5 of the smallest eps from the denominator.  With one
    gradient for all elements both states' blocks keep their largest element exactly (448 times the scale, to a
    rounding): what is left is 2^-5 and the roundings of scales."""
    from renaissance_b200 import ops
    beta2, steps = 0.999, 100
    eps = float(torch.tensor(least_eps(beta2, True) * 1.01, dtype=torch.float32))
    g = torch.full((256,), x, device="cuda")
    t = zero_states(g, True)
    plan, n = plan_of(t, 0.0, True), one(0, torch.int32)
    for _ in range(steps):
        ops.adamw_step(plan, n, 1.0, 0.9, beta2, eps)
    want = -steps * g.double() / (g.double().abs() + eps)
    off = (t["w"][0].double() - want).abs()
    assert (off <= 2.0 ** -5 * 1.01 * want.abs()).all(), float((off / want.abs()).max())


# ------------------------------------------------------------------------------------------------ huge gradients

@pytest.mark.parametrize("n", [256, 300])
@pytest.mark.parametrize("x", [2e19, -1e20, 3e38])
def test_a_finite_gradient_whose_square_overflows_spares_its_block(x, n):
    """|g| > 1.8e19 has no square in floats.  8-bit v is stored as 2^127 there: nothing becomes NaN, the other elements'
    first change is the formula's, v decays from the next step on."""
    from renaissance_b200 import ops
    g = torch.randn(n, generator=gen(1), device="cuda")
    for at in (5, n - 1):
        g[at] = x
    t = zero_states(g.clone(), True, w=0.5)
    plan, step = plan_of(t, 0.0, True), one(0, torch.int32)
    ops.adamw_step(plan, step, LR)
    tame = g.abs() < 1e3
    want = 0.5 - LR * g.double() / (g.double().abs() + EPS)
    # 1 - beta2 in floats is off by half a step of 0.999, U / 0.001 of v, half of that of the change
    assert ((t["w"][0].double() - want).abs()[tame] <= 4 * U * 0.5 + (20 + 500) * U * LR).all()
    assert (t["w"][0][~tame] == 0.5).all()                              # v is infinite in the update itself
    value = lambda: t["v"][0].float().double() * t["vs"][0].repeat_interleave(128)[:n].double()
    assert (t["m"][0].float().abs()[~tame] == 448).all()
    last = value()
    assert (last[~tame] >= 2.0 ** 127 * 0.92).all() and (last[~tame] <= 2.0 ** 127 * (1 + 8 * U)).all()     # one code below at most
    g.fill_(1.0)
    t["g"][0].fill_(1.0)
    for _ in range(500):
        ops.adamw_step(plan, step, LR)
    assert t["w"][0].isfinite().all() and t["m"][0].float().isfinite().all() and t["v"][0].float().isfinite().all()
    assert t["ms"][0].isfinite().all() and t["vs"][0].isfinite().all()
    assert (value()[~tame] < 2.0 ** 127 * 0.9).all()                    # 0.999^500 = 0.61, stochastic codes of 1/8


def test_8bit_states_with_a_non_finite_gradient_stay_nan():
    """What saturates is the square of a finite gradient only."""
    from renaissance_b200 import ops
    for bad in (math.inf, -math.inf, math.nan):
        g = torch.ones(384, device="cuda")
        g[5], g[200] = bad, 1e20
        t = zero_states(g, True)
        ops.adamw_step(plan_of(t, 0.0, True), one(0, torch.int32), LR)
        assert t["ms"][0][0].isnan() and t["vs"][0][0].isnan()
        assert t["ms"][0][1:].isfinite().all() and t["vs"][0][1:].isfinite().all()
