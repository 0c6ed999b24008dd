"""Operators for training token models with the framework, for timing and for
comparing results: the orthogonalised update of a weight matrix, and the path
of a token embedding through a K-FAC step (lookup, gradient, preconditioned
update).

``orthogonalize``  Newton-Schulz products of updates (a list of matrices):
                   X = G / (|G| + eps), then ``steps`` times
                   X = a X + (b A + c A A) X with A = X X^T;
``lookup``         rows of an embedding's weight, times a scale;
``grad``           gradient of that weight from the gradient of the rows
                   (ignored tokens give nothing);
``precondition``   kf = diag(1 / (A + damping)) grad G_inv and the momentum
                   update of an embedding's weight.
"""

import math

import torch

own = False

DEVICE = 'cuda'
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
IGNORE = -1
LR = 1e-3
MOMENTUM = 0.9
DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16,
          'float16': torch.float16}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # the smallest matrix of a network, on its own: a stem convolution
        dict(name='orthogonalize_stem', kind='orthogonalize', shapes='64x147',
             dtype='float32'),
        # one matrix of each kind that ResNet-50 has, in one call
        dict(name='orthogonalize_resnet50_kinds', kind='orthogonalize',
             shapes='64x147,64x64,64x576,256x64,128x1152,512x128,256x2304,'
                    '1024x256,512x4608,2048x512,1000x2048', dtype='float32'),
        # a wide layer of a network's body
        dict(name='orthogonalize_wide', kind='orthogonalize',
             shapes='1024x4096', dtype='float32'),
        # the largest: a square matrix
        dict(name='orthogonalize_square', kind='orthogonalize',
             shapes='4096x4096', dtype='float32'),
        # a tall layer with odd sides held in 16 bits
        dict(name='orthogonalize_tall_bf16', kind='orthogonalize',
             shapes='8191x2047', dtype='bfloat16'),
        # one token: what a generating program looks up
        dict(name='lookup_token', kind='lookup', tokens=1, vocab=32000,
             width=1024, dtype='float32', ignored=0.0),
        # a training batch, weights in 16 bits
        dict(name='lookup_batch_bf16', kind='lookup', tokens=65536,
             vocab=128000, width=2048, dtype='bfloat16', ignored=0.02),
        # a small batch over a small vocabulary
        dict(name='grad_small', kind='grad', tokens=512, vocab=8000,
             width=512, dtype='float32', ignored=0.0),
        # odd sizes, padded sequences
        dict(name='grad_odd', kind='grad', tokens=12345, vocab=32003,
             width=771, dtype='float32', ignored=0.25),
        # a large batch over a large vocabulary, gradients in 16 bits
        dict(name='grad_batch_bf16', kind='grad', tokens=65536, vocab=128000,
             width=2048, dtype='bfloat16', ignored=0.02),
        # K-FAC update of a small embedding, and of one that a batch reaches
        # a good part of
        dict(name='precondition_small', kind='precondition', tokens=512,
             vocab=8000, width=256),
        dict(name='precondition_batch', kind='precondition', tokens=32768,
             vocab=32000, width=1024),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(('orthogonalize', 'lookup', 'grad', 'precondition'))
    dtype = rng.choice(('float32', 'bfloat16'))
    if kind == 'orthogonalize':
        shapes = []
        for _ in range(rng.choice((1, 1, 2, 5))):
            rows, cols = _between(rng, 16, 4096), _between(rng, 16, 4096)
            shapes.append('%dx%d' % (rows, cols))
        # (no more work than one square matrix of the listed size)
        while sum(_products(*s) for s in _sizes(shapes)) > _products(4096, 4096):
            shapes.pop()
        return dict(kind=kind, shapes=','.join(shapes), dtype=dtype)
    if kind == 'precondition':
        return dict(kind=kind, tokens=_between(rng, 64, 32768),
                    vocab=_between(rng, 1000, 32000),
                    width=_between(rng, 32, 1024))
    return dict(kind=kind, tokens=_between(rng, 1, 65536),
                vocab=_between(rng, 1000, 128000),
                width=_between(rng, 32, 2048), dtype=dtype,
                ignored=rng.choice((0.0, 0.1, 0.5)))


def _sizes(shapes):
    return [tuple(int(v) for v in s.split('x')) for s in shapes]


def _products(rows, cols):
    """Multiply-adds, twice, of one Newton-Schulz step; the two symmetric
    products need one triangle."""
    r, c = min(rows, cols), max(rows, cols)
    return r * (r + 1) * c + r * (r + 1) * r + 2 * r * r * c


# ------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _update(g, rows, cols, dtype):
    """A momentum buffer: a part of low rank that the batches agree on, noise,
    and rows and columns of different sizes."""
    rank = max(1, min(rows, cols) // 16)
    x = torch.randn((rows, cols), device=DEVICE, generator=g)
    u = torch.randn((rows, rank), device=DEVICE, generator=g)
    v = torch.randn((rank, cols), device=DEVICE, generator=g)
    x = x + (u @ v) / rank ** 0.5
    x = x * torch.exp(0.3 * torch.randn((rows, 1), device=DEVICE, generator=g))
    x = x * torch.exp(0.3 * torch.randn((1, cols), device=DEVICE, generator=g))
    return (1e-3 * x).to(dtype)


def _shares(vocab):
    """How often each token occurs: the frequent ones come first."""
    p = 1.0 / (torch.arange(vocab, dtype=torch.float64) + 2.7)
    return p / p.sum()


def _tokens(g, tokens, vocab, ignored):
    edges = torch.cumsum(_shares(vocab), 0).to(DEVICE)
    u = torch.rand(tokens, device=DEVICE, generator=g, dtype=torch.float64)
    ids = torch.searchsorted(edges, u).clamp_(max=vocab - 1)
    if ignored:
        drop = torch.rand(tokens, device=DEVICE, generator=g) < ignored
        ids = torch.where(drop, torch.full_like(ids, IGNORE), ids)
    return ids


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    kind = case['kind']
    if kind == 'orthogonalize':
        s['x'] = [_update(g, r, c, DTYPES[case['dtype']])
                  for r, c in _sizes(case['shapes'].split(','))]
        return s
    vocab, width = case['vocab'], case['width']
    s['ids'] = _tokens(g, case['tokens'], vocab, case.get('ignored', 0.0))
    s['scale'] = width ** 0.5
    if kind == 'lookup':
        s['weight'] = (torch.randn((vocab, width), device=DEVICE, generator=g)
                       / width ** 0.5).to(DTYPES[case['dtype']])
    elif kind == 'grad':
        s['gy'] = (torch.randn((case['tokens'], width), device=DEVICE,
                               generator=g) / case['tokens']).to(
                                   DTYPES[case['dtype']])
    else:
        # gradient rows of the tokens that occurred; factors of earlier
        # batches too, so that every token has some weight in A
        n = case['tokens']
        hit = torch.zeros(vocab, dtype=torch.bool, device=DEVICE)
        hit[s['ids']] = True
        s['grad'] = torch.where(
            hit[:, None], torch.randn((vocab, width), device=DEVICE,
                                      generator=g) / n,
            torch.zeros((), device=DEVICE))
        counts = torch.bincount(s['ids'], minlength=vocab).float() / n
        s['A'] = 0.1 * counts + 0.9 * _shares(vocab).float().to(DEVICE)
        x = torch.randn((2 * width, width), device=DEVICE, generator=g)
        G = (x.T @ x).double() / (2 * width)
        G.diagonal().add_(1e-2)
        G_inv = torch.linalg.inv(G).float()
        s['G_inv'] = 0.5 * (G_inv + G_inv.T)
        s['damping'] = torch.full((1,), 1e-4, device=DEVICE)
        s['param'] = torch.randn((vocab, width), device=DEVICE, generator=g)
        s['mom'] = 1e-3 * torch.randn((vocab, width), device=DEVICE,
                                      generator=g)
    return s


# --------------------------------------------------------------------- runs

def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state['kind']](state)


def _run_own(s):
    from chainerkfac_b200 import ops
    kind = s['kind']
    if kind == 'orthogonalize':
        return ops.orthogonalize(s['x'], steps=STEPS,
                                 coefficients=COEFFICIENTS, eps=EPS)
    if kind == 'lookup':
        return ops.embedding(s['weight'], s['ids'], scale=s['scale'],
                             ignore_label=IGNORE)
    if kind == 'grad':
        order = ops.TokenOrder(s['ids'], s['vocab'], ignore_label=IGNORE)
        return ops.embedding_grad(s['gy'], order, scale=s['scale'])
    kf = ops.precondition_embedding(
        s['G_inv'], s['A'], s['damping'], s['grad'], param=s['param'],
        mom=s['mom'], lr=LR, momentum=MOMENTUM)
    return kf, s['param'], s['mom']


def _plain_orthogonalize(s):
    a, b, c = COEFFICIENTS
    out = []
    for g in s['x']:
        x = g.float()
        x = x / (x.double().square().sum().sqrt() + EPS).float()
        tall = x.shape[0] > x.shape[1]
        x = x.T if tall else x
        for _ in range(STEPS):
            gram = x @ x.T
            x = a * x + (b * gram + c * (gram @ gram)) @ x
        out.append((x.T if tall else x).contiguous().to(g.dtype))
    return out


def _plain_lookup(s):
    w, ids = s['weight'], s['ids']
    rows = w[ids.clamp(min=0)].float() * s['scale']
    return (rows * (ids != IGNORE)[:, None]).to(w.dtype)


def _plain_grad(s):
    gy, ids = s['gy'], s['ids']
    rows = gy.float() * (ids != IGNORE)[:, None]
    out = torch.zeros((s['vocab'], gy.shape[1]), device=gy.device)
    out.index_add_(0, ids.clamp(min=0), rows)
    return (out * s['scale']).to(gy.dtype)


def _plain_precondition(s):
    kf = (s['grad'] @ s['G_inv']) / (s['A'] + s['damping'])[:, None]
    s['mom'].mul_(MOMENTUM).sub_(LR * kf)
    s['param'].add_(s['mom'])
    return kf, s['param'], s['mom']


_PLAIN = {'orthogonalize': _plain_orthogonalize, 'lookup': _plain_lookup,
          'grad': _plain_grad, 'precondition': _plain_precondition}


# -------------------------------------------------------- results in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    kind = case['kind']
    if kind == 'orthogonalize':
        return [_exact_orthogonalize(x) for x in s['x']]
    if kind == 'lookup':
        out = torch.zeros((case['tokens'], case['width']),
                          dtype=torch.float64, device=DEVICE)
        at = (s['ids'] != IGNORE).nonzero().flatten()
        out[at] = s['scale'] * s['weight'].index_select(
            0, s['ids'][at]).double()
        return out
    if kind == 'grad':
        # running sums along the sorted tokens, taken apart at their ends
        ids, at = torch.sort(s['ids'])
        total = torch.cumsum(s['gy'][at].double(), 0)
        total = torch.cat((torch.zeros_like(total[:1]), total))
        v = torch.arange(case['vocab'], device=DEVICE)
        lo, hi = torch.searchsorted(ids, v), torch.searchsorted(ids, v, right=True)
        return s['scale'] * (total[hi] - total[lo])
    grad, G_inv = s['grad'].double(), s['G_inv'].double()
    d = 1.0 / (s['A'].double() + s['damping'].double())
    kf = torch.einsum('vi,v,ij->vj', grad, d, G_inv)
    mom = MOMENTUM * s['mom'].double() - LR * kf
    return kf, s['param'].double() + mom, mom


def _exact_orthogonalize(g):
    """The polynomial of the singular values, by the eigenvectors of X X^T:
    every step multiplies a singular value t by a + b t^2 + c t^4."""
    a, b, c = COEFFICIENTS
    x = g.double()
    x = x / (torch.linalg.matrix_norm(x) + EPS)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    t2, u = torch.linalg.eigh(x @ x.T)
    t2 = t2.clamp(min=0)
    gain = torch.ones_like(t2)
    for _ in range(STEPS):
        now = t2 * gain * gain
        gain = gain * (a + now * (b + now * c))
    out = u @ (gain[:, None] * (u.T @ x))
    return (out.T if tall else out).contiguous()


# --------------------------------------------------------------------- work

def _distinct(tokens, vocab):
    """Expected number of different tokens among so many."""
    p = _shares(vocab)
    return float((1.0 - torch.exp(tokens * torch.log1p(-p))).sum())


def work(case):
    kind = case['kind']
    size = 2 if case.get('dtype', 'float32') != 'float32' else 4
    if kind == 'orthogonalize':
        sizes = _sizes(case['shapes'].split(','))
        return {'bytes': 2 * size * sum(r * c for r, c in sizes),
                'flops': STEPS * sum(_products(r, c) for r, c in sizes)}
    n, vocab, width = case['tokens'], case['vocab'], case['width']
    live = n * (1.0 - case.get('ignored', 0.0))
    if kind == 'lookup':
        rows = _distinct(live, vocab)
        return {'bytes': 8 * n + size * width * (rows + n),
                'flops': live * width}
    if kind == 'grad':
        return {'bytes': 8 * n + size * width * (live + vocab),
                'flops': live * width}
    rows = _distinct(n, vocab)
    # gradient in; kf out; velocity and weight in and out
    return {'bytes': 4 * (6 * vocab * width + width * width + vocab),
            'flops': 2 * rows * width * width + 5 * vocab * width}
