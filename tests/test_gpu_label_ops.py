"""Label-vocabulary operators on the HIP path against 64 bits (bounds derived in label_cases.py)."""
import gc
import math

import numpy as np
import pytest
import torch

import label_cases as C
from oracle import label_ref as R
from shape_based_object_detection_amd import core
from shape_based_object_detection_amd.operators.Embedding import ScaledEmbedding, scaled_embedding
from shape_based_object_detection_amd.operators.Logits import process_logits
from shape_based_object_detection_amd.operators.Loss import topk_distill_loss

pytestmark = pytest.mark.gpu
DEV = 'cuda'
DT = pytest.mark.parametrize('dt', list(C.DTYPES.values()), ids=list(C.DTYPES))
TAIL = pytest.mark.parametrize('tail', [False, True], ids=['top', 'bucket'])


def dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def run_distill(x, ids, top, lse, w=None, T=1.0, reduction='mean', upstream=None):
    x = x.detach().requires_grad_(True)
    loss = topk_distill_loss(x, ids, top, lse, w, T, reduction)
    return loss, torch.autograd.grad(loss, x, upstream)[0]


# ------------------------------------------------------------------------------------------------ distillation
@DT
@TAIL
@pytest.mark.parametrize('n,v,k', [(1, 1, 1), (1, 2, 1), (3, 7, 7), (65, 21, 5), (257, 33, 8), (5, 64, 64), (9, 91, 1),
                                   (4, 255, 16), (6, 513, 100), (3, 1203, 16), (2, 1024, 1024), (3, 2048, 33),
                                   (2, 2049, 20), (3, 8191, 64), (2, 8193, 64), (2, 16385, 1000), (1, 40000, 3),
                                   (2, 50001, 100), (1, 131072, 64), (1, 200003, 50), (300, 40003, 30), (258, 61433, 7),
                                   (2, 100003, 60), (261, 70001, 1024), (259, 131070, 9),
                                   (2, 65536, 65)])
def test_distill_sizes(dt, tail, n, v, k):
    x, ids, top, lse = dev(*C.distill_inputs(n, v, k, dt, 7 * n + v + k, tail, wide=v % 2 == 0))
    loss, grad = run_distill(x, ids, top, lse, T=1.5)
    C.check_distill(loss, grad, x, ids, top, lse, None, 1.5, 'mean')


@DT
@TAIL
@pytest.mark.parametrize('v', [21, 1203, 33000, 140001])
@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
def test_distill_odd_rows(dt, tail, v, reduction):
    """Weights, repeated and absent entries, masked and dead rows, NaN where nothing may read it."""
    n, k = 14, 6
    x, ids, top, lse = C.distill_inputs(n, v, k, dt, v, tail)
    low = torch.finfo(dt).min
    ids[1] = -1                                # no entry
    ids[2, 2:] = v + 5
    ids[3] = ids[3, 0]                         # one label only, six times
    ids[4, 4] = ids[4, 1]
    x[5] = -math.inf                           # nothing left by the student's mask
    x[6, torch.randperm(v)[:v // 2]] = -math.inf
    x[6, ids[6]] = 1.0
    x[7] = low                                 # masked by the type's lowest value
    x[7, ids[7, 0]] = 0.0
    x[8] = low
    top[9, 1:] = -math.inf                     # a teacher that is sure
    x[10, :] = -math.inf                       # the student allows the kept labels alone
    x[10, ids[10]] = 0.5
    if tail:
        lse[10] = torch.logsumexp(top[10].float() / 2.0, 0) - 1e-3
    x[11, 0] = math.nan                        # weight 0: not read
    top[11, 0] = math.nan
    w = torch.rand(n) + 0.1
    w[11] = w[12] = 0
    x[13, ids[13, 0]] = 60.0                   # sure of a kept label: the others' mass is below 2^-80
    x, ids, top, lse, w = dev(x, ids, top, lse, w)
    up = torch.rand(n, device=DEV) if reduction == 'none' else torch.tensor(0.75, device=DEV)
    loss, grad = run_distill(x, ids, top, lse, w, 2.0, reduction, up)
    C.check_distill(loss, grad, x, ids, top, lse, w, 2.0, reduction, up)
    assert torch.all(grad[[1, 5] if not tail else [5]] == 0) and torch.all(grad[[11, 12]] == 0)


@DT
@pytest.mark.parametrize('v', [13, 700, 9001, 140001])
def test_distill_values_that_are_not_finite(dt, v):
    """A live row's NaN or +inf comes out as NaN; a label the student forbids but the teacher keeps as an infinite loss."""
    x, ids, top, _ = dev(*C.distill_inputs(4, v, 3, dt, 5))
    x[0, (int(ids[0].max()) + 1) % v] = math.nan
    x[1, 4] = math.inf
    x[2, ids[2, 0]] = -math.inf
    loss, grad = run_distill(x, ids, top, None, reduction='none', upstream=torch.ones(4, device=DEV))
    assert torch.isnan(loss[:2]).all() and loss[2] == math.inf and torch.isfinite(loss[3])
    assert torch.isnan(grad[:2]).any(1).all() and torch.isfinite(grad[2:]).all()
    x, ids, top, _ = dev(*C.distill_inputs(1, v, 3, dt, 6))
    x[:] = math.nan
    assert torch.isnan(run_distill(x, ids, top, None)[0])


@DT
@TAIL
@pytest.mark.parametrize('v', [21, 1203, 20001, 133001])
@pytest.mark.parametrize('extra,offset', [(0, 1), (3, 0), (5, 3), (64, 8)])
def test_distill_strides(dt, tail, v, extra, offset):
    """Rows of a padded table that start anywhere; nothing outside them is read or written."""
    n, k = 5, 4
    x, ids, top, lse = dev(*C.distill_inputs(n, v, k, dt, 3, tail))
    base = torch.full((n * (v + extra) + offset + 7,), math.nan, dtype=dt, device=DEV)
    view = base[offset:offset + n * (v + extra)].view(n, v + extra)[:, :v]
    view.copy_(x)
    loss, grad = run_distill(view, ids, top, lse, T=2.0)
    C.check_distill(loss, grad, x, ids, top, lse, None, 2.0, 'mean')
    t = x.t().contiguous().t()   # columns contiguous instead of rows
    loss, grad = run_distill(t, ids, top, lse, T=2.0)
    C.check_distill(loss, grad, x, ids, top, lse, None, 2.0, 'mean')


@DT
@pytest.mark.parametrize('v', [21, 5003, 140001])
def test_distill_backward_forms(dt, v):
    """Upstream 1, unit_grad, another factor, a retained graph used twice, no gradient: the same numbers."""
    x, ids, top, lse = dev(*C.distill_inputs(33, v, 5, dt, 11, True))
    x.requires_grad_(True)
    loss = topk_distill_loss(x, ids, top, lse, reduction='sum')
    g1, = torch.autograd.grad(loss, x, retain_graph=True)
    g1 = g1.clone()
    g2, = torch.autograd.grad(loss, x, retain_graph=True)
    assert torch.equal(g1, g2)
    g3, = torch.autograd.grad(loss * 4.0, x)           # a power of two: exact
    C.check_distill(loss, g3, x, ids, top, lse, None, 1.0, 'sum', 4.0)
    loss = topk_distill_loss(x, ids, top, lse, reduction='sum')
    g4, = torch.autograd.grad(loss, x, core.unit_grad(x.device))
    assert torch.equal(g1, g4)
    C.check_distill(loss, g1, x, ids, top, lse, None, 1.0, 'sum')
    with torch.no_grad():
        assert torch.equal(topk_distill_loss(x, ids, top, lse, reduction='sum'), loss)
    x.grad = None
    (topk_distill_loss(x[3:9].view(2, 3, v), ids[3:9].view(2, 3, 5), top[3:9].view(2, 3, 5), lse[3:9].view(2, 3),
                       reduction='none').sum() * 2).backward()
    assert torch.all(x.grad[:3] == 0) and torch.all(x.grad[9:] == 0)
    assert torch.allclose(x.grad[3:9].float(), 2 * g1[3:9].float(), rtol=4 * C.half_step(dt), atol=1e-6)


@DT
@pytest.mark.parametrize('v', [700, 30011, 90001, 140001])
def test_distill_bucket_that_holds_nearly_all(dt, v):
    """Kept labels with little mass on both sides: rest and q_o are 1 but for it, and the loss is far below the rounding
    of 1.  It is off by what its terms are, each a share P (teacher) or Q (student) of the mass."""
    n, k, T = 6, 4, 4.0
    x, ids, top, lse = C.distill_inputs(n, v, k, dt, 21, True, spread=1.0)
    top = (0.2 * top.float()).to(dt)
    lse = torch.full((n,), 11.0)
    loss, grad = run_distill(*dev(x, ids, top, lse), T=T, reduction='none', upstream=torch.ones(n, device=DEV))
    want, gwant, _ = R.distill(x.double().numpy(), ids.numpy(), top.double().numpy(), lse.double().numpy(), None, T, 'none')
    z = x.double().numpy() / T
    q = np.exp(z - z.max(1, keepdims=True))
    q /= q.sum(1, keepdims=True)
    P = np.exp(top.double().numpy() / T - 11.0).sum(1)
    Q = np.take_along_axis(q, ids.numpy(), 1).sum(1)
    A, B = np.ptp(z, axis=1), 11.0 + np.abs(top.double().numpy()).max(1) / T
    rel = C.STEP * (105 + 4 * A + 4 * B + k + 4 * math.log(v + 1.0))
    assert (P < 1e-3).all() and (Q < 0.02).all()
    assert np.all(np.abs(loss.detach().double().cpu().numpy() - want) <= T * T * rel * (2 + A + B) * 2 * (P + Q) + C.STEP * want)
    # others: share (P - Q), each of P and Q off by rel of itself
    tol = C.half_step(dt) * 1.001 * np.abs(gwant) + C.smallest(dt) + T * rel[:, None] * 4 * (np.abs(gwant) / T + q * (P + Q)[:, None])
    assert np.all(np.abs(grad.double().cpu().numpy() - gwant) <= tol)


def test_distill_half_gradients_do_not_underflow():
    """Half precision's mean over many rows is below its smallest value until the loss scale reaches it."""
    x, ids, top, _ = dev(*C.distill_inputs(2048, 640, 4, torch.float16, 2, spread=0.1))
    up = torch.tensor(65536.0, device=DEV)
    loss, grad = run_distill(x, ids, top, None, upstream=up)
    C.check_distill(loss, grad, x, ids, top, None, None, 1.0, 'mean', up)
    assert (grad != 0).all()


def test_distill_no_rows_and_no_weight():
    x, ids, top, _ = dev(*C.distill_inputs(4, 9, 2, torch.float32, 0))
    for red in ('mean', 'sum', 'none'):
        e = x[:0].clone().requires_grad_(True)
        loss = topk_distill_loss(e, ids[:0], top[:0], reduction=red)
        assert loss.shape == ((0,) if red == 'none' else ()) and loss.detach().sum() == 0
        assert torch.autograd.grad(loss.sum(), e)[0].shape == (0, 9)
    loss, grad = run_distill(x, ids, top, None, torch.zeros(4, device=DEV))
    assert loss == 0 and torch.all(grad == 0)


def test_distill_same_bits_every_time():
    x, ids, top, lse = dev(*C.distill_inputs(300, 20011, 40, torch.bfloat16, 4, True))
    ids[:, 7] = ids[:, 3]
    a, b = run_distill(x, ids, top, lse), run_distill(x, ids, top, lse)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------------------------------------ logits
def words_of(ok):
    n, v = ok.shape
    m = torch.nn.functional.pad(ok, (0, -v % 32)).view(n, -1, 32).long()
    return (m << torch.arange(32)).sum(2).to(torch.int32)


def logits_inputs(n, v, length, dt, seed, m=5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, v, generator=g) * 4).to(dt)
    hist = torch.randint(-1, v + 2, (n, length), generator=g)
    if length:
        hist[:, ::3] = hist[:, :1].clone()   # one label many times
    lens = torch.randint(-1, length + 3, (n,), generator=g)
    prompt = torch.randint(-1, length + 2, (n,), generator=g)
    rep, pre, freq = 0.5 + torch.rand(n, generator=g) * 1.5, torch.randn(n, generator=g), torch.rand(n, generator=g)
    bias = torch.randn(v, generator=g)
    bi = torch.randint(-1, v + 1, (n, m), generator=g)
    if m > 3:
        bi[:, 3] = bi[:, 0]
    bv = torch.randn(n, m, generator=g)
    ok = torch.rand(n, v, generator=g) < 0.6
    ok[-1] = False
    return x, hist, lens, prompt, rep, pre, freq, bias, bi, bv, ok


@DT
@pytest.mark.parametrize('n,v,length,m', [(1, 1, 0, 0), (1, 1, 1, 1), (3, 7, 5, 4), (65, 21, 40, 5), (2, 33, 1, 2),
                                          (4, 1203, 300, 9), (2, 4095, 64, 5), (3, 4097, 5000, 300), (2, 32000, 300, 5),
                                          (3, 50001, 1025, 64), (1, 131072, 20000, 17)])
@pytest.mark.parametrize('kind', ['bits', 'bool', 'plain'])
def test_logits_sizes(dt, n, v, length, m, kind):
    x, hist, lens, prompt, rep, pre, freq, bias, bi, bv, ok = logits_inputs(n, v, length, dt, v + length, m)
    if kind == 'plain':
        kw = dict(history=hist[0].int(), repetition=1.25, presence=0.5, frequency=0.125, bias=bias.to(dt))
        allowed, okn = None, None
    else:
        kw = dict(history=hist, history_len=lens, prompt_len=prompt.int(), repetition=rep, presence=pre, frequency=freq,
                  bias=bias.expand(n, v) if kind == 'bool' else None, bias_ids=bi, bias_values=bv)
        allowed, okn = (ok if kind == 'bool' else words_of(ok)), ok.numpy()
    ref = {a: (t.float().numpy() if torch.is_tensor(t) and t.is_floating_point() else t.numpy() if torch.is_tensor(t) else t)
           for a, t in kw.items()}
    want, mag = R.process_logits(x.double().numpy(), allowed=okn, **ref)
    xd = x.to(DEV)
    kd = {a: t.to(DEV) if torch.is_tensor(t) else t for a, t in kw.items()}
    allowed = None if allowed is None else allowed.to(DEV)
    got = process_logits(xd, allowed=allowed, **kd)
    C.check_logits(got, want, mag, dt, 3 + m)
    assert torch.equal(xd, x.to(DEV))
    assert process_logits(xd, allowed=allowed, out=xd, **kd) is xd
    assert torch.equal(xd, got) or torch.equal(xd.isnan(), got.isnan())


@DT
def test_logits_special_values(dt):
    """NaN and infinities in masked and unmasked places, one mask row for all, a mask of the type's lowest value as bias."""
    x = torch.randn(3, 70).to(dt)
    x[0, 3], x[1, 4], x[2, 5], x[0, 6] = math.nan, math.inf, -math.inf, math.nan
    ok = torch.ones(70, dtype=torch.bool)
    ok[3] = ok[4] = False
    bias = torch.zeros(70).to(dt)
    bias[8] = -math.inf
    bias[9] = torch.finfo(dt).min
    hist = torch.tensor([[3, 5, 6, 9]]).expand(3, 4)
    kw = dict(history=hist, repetition=2.0, presence=1.0, bias=bias)
    want, mag = R.process_logits(x.double().numpy(), hist.numpy(), repetition=2.0, presence=1.0,
                                 bias=bias.double().numpy(), allowed=ok.numpy())
    for allowed in (ok, words_of(ok[None])[0]):
        got = process_logits(x.to(DEV), allowed=allowed.to(DEV), **{a: t.to(DEV) if torch.is_tensor(t) else t for a, t in kw.items()})
        C.check_logits(got, want, np.where(np.isfinite(mag), mag, 0), dt, 4)
        assert torch.all(got[:, 3] == -math.inf) and torch.all(got[:, 4] == -math.inf) and got[0, 6].isnan()


@DT
@pytest.mark.parametrize('v', [50, 4100])
@pytest.mark.parametrize('offset,pad', [(0, 5), (1, 0), (3, 7)])
def test_logits_strides_and_out(dt, v, offset, pad):
    x, hist, lens, prompt, rep, pre, freq, bias, bi, bv, ok = logits_inputs(4, v, 30, dt, 1)
    full = process_logits(*dev(x, hist, lens, prompt, rep, pre, freq, bias, bi, bv, ok))
    buf = torch.full((4 * (v + pad) + offset,), 7.0, dtype=dt, device=DEV)
    view = buf[offset:].view(4, v + pad)[:, :v]
    view.copy_(x)
    wide = torch.zeros(4, 2 * v, dtype=torch.bool, device=DEV)
    wide[:, ::2] = ok.to(DEV)
    args = dev(hist, lens, prompt, rep, pre, freq, bias, bi, bv)
    hw = torch.full((4, 44), 3, dtype=torch.int64, device=DEV)
    hw[:, :30] = args[0]
    got = process_logits(view, hw[:, :30], *args[1:], wide[:, ::2])
    assert torch.equal(got, full)
    fresh = torch.full((4, v + 3), 5.0, dtype=dt, device=DEV)   # an out whose rows lie otherwise
    process_logits(view, *args, ok.to(DEV), out=fresh[:, :v])
    assert torch.equal(fresh[:, :v], full) and torch.all(fresh[:, v:] == 5)
    process_logits(view, *args, ok.to(DEV), out=view)
    assert torch.equal(view, full)
    if pad:
        assert torch.all(buf[offset:].view(4, v + pad)[:, v:] == 7)
    with pytest.raises(ValueError, match='overlaps'):
        process_logits(view[:2], out=view[1:3])
    with pytest.raises(ValueError, match='contiguous'):
        process_logits(x.to(DEV), out=torch.empty(v, 4, dtype=dt, device=DEV).t())


# ------------------------------------------------------------------------------------------------ embedding
@DT
@pytest.mark.parametrize('n,v,d', [(0, 3, 4), (1, 1, 1), (5, 3, 7), (32, 50, 8), (100, 2, 33), (64, 1000, 129), (700, 21, 256),
                                   (1025, 300, 100), (3, 5000, 4096), (5000, 5, 17), (20000, 700, 24), (70000, 3, 8),
                                   (4096, 131072, 8), (130, 8, 8192)])
@pytest.mark.parametrize('wide', [True, False], ids=['i64', 'i32'])
def test_embedding_sizes(dt, n, v, d, wide):
    g = torch.Generator().manual_seed(n + v + d)
    ids = (torch.rand(n, generator=g) ** 2 * (v + 1)).long() - (1 if n > 3 else 0)   # some absent, most low
    ids = ids.clamp(max=v) if wide else ids.clamp(max=v).int()
    w = torch.randn(v, d, generator=g).to(dt)
    go = torch.randn(n, d, generator=g).to(dt)
    wd = w.to(DEV).requires_grad_(True)
    out = scaled_embedding(ids.to(DEV), wd, 1.7, 0 if n > 3 else None)
    grad, = torch.autograd.grad(out, wd, go.to(DEV))
    there = (ids >= 0) & (ids < v)
    # one rounding of the product, through float32 or not: half a step of dt and one of float32 hold both
    want = (w[ids.long().clamp(0, v - 1)].double() * float(np.float32(1.7))).masked_fill(~there[:, None], 0)
    assert torch.all((out.cpu().double() - want).abs() <= (C.half_step(dt) + C.STEP) * want.abs() + C.smallest(dt))
    C.check_embedding_grad(grad, ids, go, v, 1.7, 0 if n > 3 else -1)
    again, = torch.autograd.grad(scaled_embedding(ids.to(DEV), wd, 1.7, 0 if n > 3 else None), wd, go.to(DEV))
    assert torch.equal(grad, again)


@DT
def test_embedding_forms(dt):
    """Leading shapes, a table and a gradient that start off a 16-byte boundary, an expanded gradient, the module."""
    v, d = 40, 24
    store = torch.randn(v * d + 3, device=DEV).to(dt)
    table = store[3:].view(v, d).requires_grad_(True)
    ids = torch.randint(0, v, (3, 4, 5), device=DEV)
    out = scaled_embedding(ids, table, 0.5, -1)
    assert out.shape == (3, 4, 5, d) and torch.equal(out, table[ids] * 0.5)
    one = torch.randn(d, device=DEV).to(dt)
    grad, = torch.autograd.grad(out, table, one.expand(3, 4, 5, d))
    C.check_embedding_grad(grad, ids, one.expand(60, d), v, 0.5, v - 1)
    m = ScaledEmbedding(v, d, padding_idx=7, device=DEV, dtype=dt)
    m(torch.full((6,), 7, device=DEV)).sum().backward()
    assert torch.all(m.weight.grad == 0) and torch.all(m.weight[7] == 0)
    assert scaled_embedding(ids[:0], table).shape == (0, 4, 5, d)


# ------------------------------------------------------------------------------------------------ together
def test_label_by_label_training_and_answering():
    """A label decoder as it is used: its queries looked up, the next label's logits learnt from a teacher's top ones
    through the same table, then answered under a grammar, the answers looked up again."""
    torch.manual_seed(0)
    v, d, n, k = 1001, 64, 48, 8
    table = ScaledEmbedding(v, d, device=DEV)
    ids = torch.randint(0, v, (n,), device=DEV)
    teacher = torch.randn(n, v, device=DEV) * 3
    ok = torch.rand(n, v, device=DEV) < 0.7
    seen = process_logits(teacher, ids[:, None], repetition=1.2, allowed=ok)
    top, tid = seen.topk(k, 1)
    lse = torch.logsumexp(seen / 2.0, 1)
    loss = topk_distill_loss(table(ids) @ table.weight.t(), tid, top, lse, temperature=2.0)
    loss.backward()
    w = table.weight.detach().double().requires_grad_(True)
    q = torch.log_softmax((w[ids] * table.scale) @ w.t() / 2.0, 1)
    lp = top.double() / 2.0 - lse.double()[:, None]
    rest = 1 - lp.exp().sum(1)
    kl = (lp.exp() * (lp - q.gather(1, tid))).sum(1)
    kl = kl + rest * (rest.log() - torch.logsumexp(q.scatter(1, tid, -math.inf), 1))
    ref = 4.0 * kl.mean()
    ref.backward()
    # float32 products of 64 terms and sums of 1,001 between the two: 2e-5 of the largest value holds them
    assert abs(float(loss) - float(ref)) < 2e-5 * abs(float(ref))
    assert (table.weight.grad.double() - w.grad).abs().max() < 2e-5 * w.grad.abs().max()
    with torch.no_grad():
        hist = torch.full((n, 6), -1, dtype=torch.int64, device=DEV)
        hist[:, 0] = ids
        last = ids
        for step in range(1, 6):
            logits = table(last) @ table.weight.t()
            last = process_logits(logits, hist, repetition=1.0, presence=1e6, allowed=ok, out=logits).argmax(1)
            assert ok.gather(1, last[:, None]).all() and not (hist == last[:, None]).any()
            hist[:, step] = last


@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16, torch.float16], ids=['f32', 'bf16', 'f16'])
def test_captured_steps_equal_eager(dt):
    """A training step and an answering step captured into one graph each, replayed with new inputs and eager work
    and synchronisations between the replays."""
    v, d, n, k = 3001, 48, 40, 6
    s = torch.cuda.Stream()
    w = (torch.randn(v, d, device=DEV) * 0.2).to(dt)
    ids = torch.zeros(n, dtype=torch.int64, device=DEV)
    x = torch.zeros(n, v, dtype=dt, device=DEV)
    tid = torch.zeros(n, k, dtype=torch.int64, device=DEV)
    top, lse = torch.zeros(n, k, dtype=dt, device=DEV), torch.zeros(n, device=DEV)
    up = torch.tensor(8.0, device=DEV)
    go = torch.zeros(n, d, dtype=dt, device=DEV)

    def step():
        xx, ww = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = topk_distill_loss(xx, tid, top, lse, temperature=2.0)
        gx, = torch.autograd.grad(loss, xx, up)
        out = scaled_embedding(ids, ww, 3.0)
        gw, = torch.autograd.grad(out, ww, go)
        return loss.detach(), gx, out.detach(), gw, process_logits(x, tid, presence=0.5, repetition=1.5)

    def fill(seed):
        a = C.distill_inputs(n, v, k, dt, seed, True)
        for t, b in zip((x, tid, top, lse), a):
            t.copy_(b)
        ids.copy_(torch.randint(0, v, (n,)))
        go.copy_(torch.randn(n, d))
        up.fill_(float(seed % 2) * 7 + 1)

    fill(0)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = step()
    for seed in (1, 2, 3, 4):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_capture_is_refused_while_an_eager_graph_holds_the_leaves():
    """(Its captured backward pass would join the eager graph's stream; only forward calls are made here.)"""
    x, tid, top, _ = dev(*C.distill_inputs(6, 40, 3, torch.float32, 2, True))
    table = torch.randn(9, 40, device=DEV).requires_grad_(True)
    leaf = x.clone().requires_grad_(True)
    ids = torch.arange(6, device=DEV)
    calls = {'embed': lambda: scaled_embedding(ids, table, 2.0), 'leaf': lambda: topk_distill_loss(leaf, tid, top),
             'network': lambda: topk_distill_loss(table[:6] * 2.0, tid, top)}
    s = torch.cuda.Stream()
    for name, call in calls.items():
        held = call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            with pytest.raises(RuntimeError, match='release its result first'):
                call()
            with torch.no_grad():
                again = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, held.detach()), name
        del held
        gc.collect()
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
            call()


def test_other_streams():
    """Calls on several streams at once hold their own scratch memory."""
    sets = [dev(*C.distill_inputs(64, 30011, 16, torch.bfloat16, i, True)) for i in range(4)]
    ids = [torch.randint(0, 500, (4000,), device=DEV) for _ in sets]
    w = torch.randn(500, 64, device=DEV)
    go = torch.randn(4000, 64, device=DEV)

    def step(i):
        ww = w.detach().requires_grad_(True)
        return run_distill(*sets[i]) + torch.autograd.grad(scaled_embedding(ids[i], ww), ww, go)

    want = [step(i) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(3):
        got = []
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append(step(i))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@DT
def test_native_calls_equal_python_path(dt, monkeypatch):
    """The C++ calls (csrc/host_label.h) and core.py's give the same bits, in every form that both take."""
    from shape_based_object_detection_amd import _lib as L
    x, ids, top, lse = dev(*C.distill_inputs(24, 2600, 9, dt, 8, True))
    w = torch.rand(24, device=DEV)
    lg = [t.to(DEV) for t in logits_inputs(24, 2600, 40, dt, 2)]
    lg[2], lg[3] = lg[2].int(), lg[3].int()
    table = torch.randn(50, 12, device=DEV).to(dt).requires_grad_(True)
    tid = torch.randint(-1, 51, (6, 7), device=DEV)
    go = torch.randn(6, 7, 12, device=DEV).to(dt)

    def everything():
        got = []
        for red in ('mean', 'sum', 'none'):
            for a, b in ((None, None), (lse, None), (None, w), (lse, w)):
                for up in (1.0, 3.0):
                    u = torch.full((24,) if red == 'none' else (), up, device=DEV)
                    got += run_distill(x, ids, top, a, b, 1.5, red, u)
        xx = x.clone().requires_grad_(True)
        loss = topk_distill_loss(xx, ids, top, reduction='sum')
        got += torch.autograd.grad(loss, xx, core.unit_grad(x.device), retain_graph=True)
        got += torch.autograd.grad(loss, xx)
        g, = torch.autograd.grad(topk_distill_loss(xx, ids, top), xx, create_graph=True)
        with pytest.raises(RuntimeError, match='twice'):
            g.square().sum().backward()
        got.append(g.detach())
        got += [process_logits(*lg[:10], lg[10]), process_logits(lg[0], lg[1], presence=0.5, allowed=lg[10][0]),
                process_logits(lg[0], bias=lg[7], allowed=words_of(lg[10].cpu()).to(DEV))]
        y = lg[0].clone()
        v0 = y._version
        got.append(process_logits(y, lg[1], frequency=0.25, out=y))
        assert got[-1] is y and y._version > v0
        for pad in (None, 3, -1):
            out = scaled_embedding(tid, table, 2.5, pad)
            got += [out.detach(), torch.autograd.grad(out, table, go)[0]]
        return got

    L.lib()
    ext = L.host_ext
    assert ext is not None
    native = everything()
    assert 'DistillFn' in topk_distill_loss(x.clone().requires_grad_(True), ids, top).grad_fn.name()
    monkeypatch.setattr(L, 'host_ext', None)
    python = everything()
    assert len(native) == len(python)
    for a, b in zip(native, python):
        assert a.shape == b.shape and torch.equal(a.nan_to_num(), b.nan_to_num())


def test_devices_are_not_mixed():
    x, ids, top, _ = C.distill_inputs(2, 5, 2, torch.float32, 0)
    with pytest.raises(RuntimeError):
        topk_distill_loss(x.to(DEV), ids, top.to(DEV))
    with pytest.raises(RuntimeError):
        process_logits(x.to(DEV), bias=torch.zeros(5))
    with pytest.raises(RuntimeError):
        scaled_embedding(ids.to(DEV), x)
    with pytest.raises(TypeError):
        topk_distill_loss(x.to(DEV).double(), ids.to(DEV), top.to(DEV))
    with pytest.raises(TypeError):
        process_logits(x.to(DEV).double())
    with pytest.raises(TypeError):
        scaled_embedding(ids.to(DEV), x.to(DEV).double())
