"""Cases and plain forms of the label-vocabulary operators: what a class vocabulary takes in, learns and answers.

  distill  operators.Loss.topk_distill_loss: a student's class logits against the few top logits kept of a teacher's,
           with the gradient
  logits   operators.Logits.process_logits: penalties for repeated labels, biases and masks on the logits that a
           decoder is about to choose from
  embed    operators.Embedding.scaled_embedding: rows of a label table, scaled, and the table's gradient

``own`` picks between the plain form (elementary torch operations, 32 bits, one rounding at the end) and the
framework's calls.  ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

_DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
_BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}


def listed():
    return [
        # every anchor of a batch of 32 SSD512 images (10,248 priors, 21 classes) against five kept classes of a
        # teacher detector; anchors without an object nearby carry weight 0
        dict(name='distill anchors', op='distill', n=327936, v=21, k=5, dt='f32', tail=False, weights=True,
             reduction='mean', temperature=2.0, upstream=1.0),
        # proposals over an open vocabulary's classes, the teacher's remaining mass kept as one bucket
        dict(name='distill proposals', op='distill', n=32768, v=1203, k=16, dt='bf16', tail=True, weights=True,
             reduction='mean', temperature=1.0, upstream=1.0),
        # a training batch over an odd vocabulary in full precision
        dict(name='distill odd f32', op='distill', n=2049, v=50001, k=100, dt='f32', tail=True, weights=False,
             reduction='sum', temperature=1.5, upstream=1.0),
        # the largest: 4,096 positions over 131,072 labels
        dict(name='distill large', op='distill', n=4096, v=131072, k=64, dt='bf16', tail=False, weights=False,
             reduction='mean', temperature=1.0, upstream=1.0),
        # a few positions in half precision, its loss scaled as mixed-precision training does
        dict(name='distill few rows', op='distill', n=7, v=32003, k=20, dt='f16', tail=True, weights=False,
             reduction='mean', temperature=1.0, upstream=1024.0),
        # one sequence that answers label by label: latency counts
        dict(name='logits one row', op='logits', n=1, v=32000, length=300, dt='f32', bias='none', m=0, mask='bits',
             allowed=0.5),
        # a serving batch: ragged histories, request biases, a grammar's bit masks
        dict(name='logits batch', op='logits', n=256, v=131072, length=4096, dt='bf16', bias='sparse', m=300,
             mask='bits', allowed=0.75),
        # a bias of the class frequencies and a truth-value mask over an odd vocabulary
        dict(name='logits odd f16', op='logits', n=61, v=50001, length=1025, dt='f16', bias='dense', m=0, mask='bool',
             allowed=0.25),
        # the next label of each of 32 sequences
        dict(name='embed next', op='embed', n=32, v=131072, d=4096, dt='bf16', train=False, skew=0.0),
        # label queries of a batch of 32 images, 200 each, over 21 classes: every row of the table many times
        dict(name='embed labels', op='embed', n=6400, v=21, d=256, dt='f32', train=True, skew=0.0),
        # a prompt batch whose labels follow their frequencies
        dict(name='embed prompts', op='embed', n=8192, v=32000, d=2048, dt='bf16', train=True, skew=1.0),
        # the largest: 65,536 labels, a table of 131,072 rows
        dict(name='embed large', op='embed', n=65536, v=131072, d=4096, dt='bf16', train=True, skew=1.0),
    ]


def _log(rng, lo, hi):
    """A whole number, its logarithm spread evenly over [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['distill', 'logits', 'embed'])
    dt = rng.choice(['f32', 'bf16', 'f16'])
    wide = 2 if dt == 'f32' else 1
    if op == 'distill':
        v = _log(rng, 11, 160001)
        n = _log(rng, 1, min(300001, (1 << 27) // (v * wide)))
        return dict(op=op, n=n, v=v, k=_log(rng, 1, min(v // 2, 256)), dt=dt, tail=rng.random() < 0.5,
                    weights=rng.random() < 0.5, reduction=rng.choice(['mean', 'sum', 'none']),
                    temperature=rng.choice([0.5, 1.0, 2.0, 4.0]), upstream=rng.choice([1.0, 0.25]))
    if op == 'logits':
        v = _log(rng, 21, 160001)
        n = _log(rng, 1, min(4096, (1 << 24) // v))
        bias = rng.choice(['none', 'sparse', 'dense'])
        return dict(op=op, n=n, v=v, length=_log(rng, 1, min(8191, (1 << 20) // n)), dt=dt, bias=bias,
                    m=_log(rng, 1, min(v, 300)) if bias == 'sparse' else 0, mask=rng.choice(['none', 'bits', 'bool']),
                    allowed=rng.choice([0.02, 0.5, 0.98]))
    d = _log(rng, 8, 8191)
    v = _log(rng, 11, min(160001, (1 << 28) // (d * wide)))
    n = _log(rng, 1, min(131071, (1 << 27) // (d * wide)))
    return dict(op=op, n=n, v=v, d=d, dt=dt, train=rng.random() < 0.7, skew=rng.choice([0.0, 0.5, 1.0]))


# ------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    op = case['op']
    if op == 'distill':
        return _prepare_distill(case, g)
    return _prepare_logits(case, g) if op == 'logits' else _prepare_embed(case, g)


def _prepare_distill(c, g):
    n, v, k, dt = c['n'], c['v'], c['k'], _DT[c['dt']]
    x = torch.randn(n, v, generator=g, device='cuda', dtype=torch.float32).mul_(2.0)
    # the teacher's top classes: k different ones, spread over the vocabulary, that the student half agrees on
    u = torch.rand(n, k, generator=g, device='cuda')
    ids = ((torch.arange(k, device='cuda') + u) * (v / k)).long().clamp_(max=v - 1)
    top = 4.0 + 3.0 * torch.rand(n, k, generator=g, device='cuda')
    x.scatter_add_(1, ids, 0.5 * top)
    t = top.to(dt).float() / c['temperature']
    rest = math.log(max(v - k, 1)) + 0.3 * torch.randn(n, generator=g, device='cuda')
    lse = torch.logaddexp(torch.logsumexp(t, 1), rest) if c['tail'] else None
    w = (torch.rand(n, generator=g, device='cuda') < 0.4).float() if c['weights'] else None
    if w is not None:
        w[0] = 1.0   # a batch has at least one row to learn from
    rows = torch.rand(n, generator=g, device='cuda') if c['reduction'] == 'none' else None
    up = c['upstream'] * (torch.ones((), device='cuda') if rows is None else rows)
    return dict(c, x=x.to(dt).requires_grad_(True), ids=ids, top=top.to(dt), lse=lse, w=w, up=up)


def _bits(mask):
    """Truth values [n, v] as int32 words, label j in bit j % 32 of word j // 32."""
    n, v = mask.shape
    m = torch.nn.functional.pad(mask, (0, -v % 32)).view(n, -1, 32).long()
    return (m << torch.arange(32, device=m.device)).sum(2).to(torch.int32)


def _prepare_logits(c, g):
    n, v, length, dt = c['n'], c['v'], c['length'], _DT[c['dt']]
    x = torch.randn(n, v, generator=g, device='cuda').mul_(4.0).to(dt)
    # labels repeat: a history is drawn from the vocabulary by frequency
    hist = (torch.rand(n, length, generator=g, device='cuda') ** 3 * v).long().clamp_(max=v - 1)
    lens = (torch.rand(n, generator=g, device='cuda') * (length + 1)).int().clamp_(max=length)
    if n == 1:
        lens.fill_(length)
    prompt = (lens * torch.rand(n, generator=g, device='cuda')).int()
    rep = 1.0 + 0.5 * torch.rand(n, generator=g, device='cuda')
    pre = torch.rand(n, generator=g, device='cuda')
    freq = 0.25 * torch.rand(n, generator=g, device='cuda')
    bias = torch.randn(v, generator=g, device='cuda') if c['bias'] == 'dense' else None
    bi = bv = None
    if c['bias'] == 'sparse':
        u = torch.rand(n, c['m'], generator=g, device='cuda')
        bi = ((torch.arange(c['m'], device='cuda') + u) * (v / c['m'])).long().clamp_(max=v - 1)
        bv = 5.0 * torch.randn(n, c['m'], generator=g, device='cuda')
    mask = None
    if c['mask'] != 'none':
        # a grammar allows or forbids runs of the vocabulary more than single labels
        runs = torch.rand(n, (v + 63) // 64, generator=g, device='cuda') < c['allowed']
        mask = runs.repeat_interleave(64, dim=1)[:, :v].contiguous()
        mask = _bits(mask) if c['mask'] == 'bits' else mask
    return dict(c, x=x, hist=hist, lens=lens, prompt=prompt, rep=rep, pre=pre, freq=freq, bias_row=bias, bi=bi, bv=bv,
                allow=mask)


def _prepare_embed(c, g):
    n, v, d, dt = c['n'], c['v'], c['d'], _DT[c['dt']]
    w = torch.randn(v, d, generator=g, device='cuda', dtype=dt).mul_(0.02)
    u = torch.rand(n, generator=g, device='cuda', dtype=torch.float64)
    # skew 0: every label alike; 1: label r about as often as 1 / r
    ids = (torch.exp(u * math.log(v)) - 1.0 if c['skew'] == 1.0 else u ** (1.0 + 2.0 * c['skew']) * v)
    ids = torch.randperm(v, generator=g, device='cuda')[ids.long().clamp_(0, v - 1)]
    gout = torch.randn(n, d, generator=g, device='cuda', dtype=dt) if c['train'] else None
    return dict(c, w=w.requires_grad_(c['train']), ids=ids, gout=gout, scale=math.sqrt(d))


# ------------------------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _own(state)
    op = state['op']
    with torch.no_grad():
        if op == 'distill':
            return _plain_distill(state)
        return _plain_logits(state) if op == 'logits' else _plain_embed(state)


def _own(s):
    if s['op'] == 'distill':
        from shape_based_object_detection_amd.operators.Loss import topk_distill_loss
        loss = topk_distill_loss(s['x'], s['ids'], s['top'], teacher_lse=s['lse'], weights=s['w'],
                                 temperature=s['temperature'], reduction=s['reduction'])
        grad, = torch.autograd.grad(loss, s['x'], s['up'])
        return loss.detach(), grad
    if s['op'] == 'logits':
        from shape_based_object_detection_amd.operators.Logits import process_logits
        return process_logits(s['x'], s['hist'], history_len=s['lens'], prompt_len=s['prompt'], repetition=s['rep'],
                              presence=s['pre'], frequency=s['freq'], bias=s['bias_row'], bias_ids=s['bi'],
                              bias_values=s['bv'], allowed=s['allow'])
    from shape_based_object_detection_amd.operators.Embedding import scaled_embedding
    out = scaled_embedding(s['ids'], s['w'], scale=s['scale'])
    if not s['train']:
        return out
    grad, = torch.autograd.grad(out, s['w'], s['gout'])
    return out.detach(), grad


def _plain_distill(s):
    T = s['temperature']
    x = s['x'].float()
    x = (x - x.amax(1, keepdim=True)) / T
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    logq = x.gather(1, s['ids']) - torch.log(total)
    t = s['top'].float() / T
    if s['lse'] is None:
        t = t - t.amax(1, keepdim=True)
        logp = t - torch.log(torch.exp(t).sum(1, keepdim=True))
        p = torch.exp(logp)
        rows = (p * (logp - logq)).sum(1)
        grad = e / total
    else:
        logp = t - s['lse'][:, None]
        p = torch.exp(logp)
        rest = (1.0 - p.sum(1, keepdim=True)).clamp(min=0.0)
        kept = e.scatter(1, s['ids'], 0.0)
        other = kept.sum(1, keepdim=True) / total
        logr = torch.log(rest) - torch.log(other)
        rows = (p * (logp - logq)).sum(1) + torch.where(rest > 0, rest * logr, rest)[:, 0]
        grad = kept / total * (1.0 - rest / other)
        grad.scatter_(1, s['ids'], torch.exp(logq))
    grad.scatter_add_(1, s['ids'], -p)
    rows = rows * (T * T)
    w = torch.ones_like(rows) if s['w'] is None else s['w']
    scale = w / w.sum() if s['reduction'] == 'mean' else w
    loss = scale * rows if s['reduction'] == 'none' else (scale * rows).sum()
    grad = grad * (scale * s['up'] * T)[:, None]
    return loss, grad.to(s['x'].dtype)


def _plain_logits(s):
    x = s['x'].float()
    n, v = x.shape
    place = torch.arange(s['length'], device=x.device)
    live = place < s['lens'][:, None]
    answered = live & (place >= s['prompt'][:, None])
    seen = torch.zeros(n, v, device=x.device).scatter_add_(1, s['hist'], live.float()) > 0
    count = torch.zeros(n, v, device=x.device).scatter_add_(1, s['hist'], answered.float())
    rep = s['rep'][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s['freq'][:, None] * count - s['pre'][:, None] * (count > 0)
    if s['bias_row'] is not None:
        x = x + s['bias_row']
    if s['bi'] is not None:
        x = x.scatter_add(1, s['bi'], s['bv'])
    if s['allow'] is not None:
        allow = s['allow']
        if allow.dtype != torch.bool:
            label = torch.arange(v, device=x.device)
            allow = (allow[:, label // 32] >> (label % 32)) & 1 > 0
        x = x.masked_fill(~allow, -math.inf)
    return x.to(s['x'].dtype)


def _plain_embed(s):
    out = (s['w'][s['ids']].float() * s['scale']).to(s['w'].dtype)
    if not s['train']:
        return out
    grad = torch.zeros(s['v'], s['d'], device=out.device).index_add_(0, s['ids'], s['gout'].float())
    return out, (grad * s['scale']).to(s['w'].dtype)


# ------------------------------------------------------------------------------------------------- the definition
def exact(case, seed):
    s = prepare(case, seed)
    if s['op'] == 'distill':
        return _exact_distill(s)
    with torch.no_grad():
        return _exact_logits(s) if s['op'] == 'logits' else _exact_embed(s)


def _exact_distill(s):
    """KL(teacher || student) at temperature T, times T^2, by 64-bit autograd."""
    T, ids = s['temperature'], s['ids']
    x = s['x'].detach().double().requires_grad_(True)
    logq = torch.log_softmax(x / T, 1)
    t = s['top'].double() / T
    if s['lse'] is None:
        logp = torch.log_softmax(t, 1)
        kl = (logp.exp() * (logp - logq.gather(1, ids))).sum(1)
    else:
        logp = t - s['lse'].double()[:, None]
        kl = (logp.exp() * (logp - logq.gather(1, ids))).sum(1)
        rest = 1.0 - logp.exp().sum(1)
        others = logq.scatter(1, ids, -math.inf)
        kl = kl + torch.where(rest > 0, torch.special.xlogy(rest.clamp(min=0), rest.clamp(min=1e-300))
                              - rest.clamp(min=0) * torch.logsumexp(others, 1), torch.zeros_like(rest))
    rows = T * T * kl
    if s['w'] is not None:
        rows = rows * s['w'].double()
    if s['reduction'] == 'none':
        loss = rows
    else:
        loss = rows.sum()
        if s['reduction'] == 'mean':
            loss = loss / (s['n'] if s['w'] is None else s['w'].double().sum())
    grad, = torch.autograd.grad(loss, x, s['up'].double())
    return loss.detach(), grad


def _exact_logits(s):
    x = s['x'].double()
    n, v, length = s['n'], s['v'], s['length']
    row = torch.arange(n, device=x.device)[:, None].expand(n, length)
    place = torch.arange(length, device=x.device).expand(n, length)
    live = place < s['lens'][:, None]
    late = live & (place >= s['prompt'][:, None])
    flat = row * v + s['hist']
    seen = torch.bincount(flat[live], minlength=n * v).view(n, v) > 0
    count = torch.bincount(flat[late], minlength=n * v).view(n, v).double()
    rep = s['rep'].double()[:, None]
    factor = torch.where(seen, torch.where(x > 0, 1.0 / rep, rep), torch.ones_like(x))
    x = x * factor - count * s['freq'].double()[:, None] - count.clamp(max=1) * s['pre'].double()[:, None]
    if s['bias_row'] is not None:
        x += s['bias_row'].double()
    if s['bi'] is not None:
        x.view(-1).index_add_(0, (torch.arange(n, device=x.device)[:, None] * v + s['bi']).view(-1), s['bv'].double().view(-1))
    if s['mask'] == 'bool':
        x[~s['allow']] = -math.inf
    elif s['mask'] == 'bits':
        shift = torch.arange(32, device=x.device)
        x[((s['allow'].long()[:, :, None] >> shift) % 2 == 0).view(n, -1)[:, :v]] = -math.inf
    return x


def _exact_embed(s):
    out = s['w'].detach().double().index_select(0, s['ids']) * s['scale']
    if not s['train']:
        return out
    grad = torch.zeros(s['v'], s['d'], dtype=torch.float64, device=out.device)
    grad.index_put_((s['ids'],), s['gout'].double(), accumulate=True)
    return out, grad * s['scale']


# ------------------------------------------------------------------------------------------------- the work
def work(case):
    """Bytes that one pass has to read and write, each input and output once, and its operations."""
    b = _BYTES[case['dt']]
    n, op = case['n'], case['op']
    if op == 'distill':
        v, k = case['v'], case['k']
        return {'bytes': n * (2 * v * b + k * (8 + b) + 4 * case['tail'] + 4 * case['weights']), 'flops': 6 * n * v}
    if op == 'logits':
        v = case['v']
        mask = {'none': 0, 'bits': n * ((v + 31) // 32) * 4, 'bool': n * v}[case['mask']]
        bias = {'none': 0, 'sparse': n * case['m'] * 12, 'dense': 4 * v}[case['bias']]
        return {'bytes': n * (2 * v * b + 8 * (case['length'] + 1) // 2 + 20) + mask + bias, 'flops': 6 * n * v}
    d, v = case['d'], case['v']
    r = torch.arange(v + 1, dtype=torch.float64) / v   # the labels' shares, by their ranks (_prepare_embed)
    r = torch.log1p(r * (v - 1)) / math.log(v) if case['skew'] == 1.0 else r ** (1.0 / (1.0 + 2.0 * case['skew']))
    rows = float(-torch.expm1(n * torch.log1p(-r.diff().clamp(max=1 - 1e-9))).sum())   # different labels among n
    return {'bytes': n * 8 + (rows + n) * d * b + case['train'] * (n + v) * d * b, 'flops': (1 + case['train']) * n * d}
