"""Cases and plain forms of the channels-last group norm and of the 8-bit integer product.

  gn        y = act(group_norm(x)), forward only
  gn_train  the same with its backward pass: y, dx, dgamma, dbeta
  int8      y = act(x @ w.T + bias): the rows of x quantised to 8 bits with a scale a row, w held in 8 bits with a scale an
            output channel (a 1x1 convolution over pixels, or a linear layer over tokens)
  gn_int8   group norm + activation quantised to 8-bit rows, and the product of those

Feature maps are (batch, channels, height, width) tensors in channels_last memory.
"""
import torch

own = False

TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}
SIZE = {'fp16': 2, 'bf16': 2, 'fp32': 4}
EPS = 1e-5
SLOPE = 0.1  # LeakyReLU slope of the framework's convolution blocks
ZERO_ROW = 2.0 ** -120  # a row whose largest magnitude is below this counts as a row of zeros


def _gn(op, name, dtype, batch, height, width, channels, groups, act, cout=0):
    c = {'op': op, 'dtype': dtype, 'batch': batch, 'height': height, 'width': width, 'channels': channels, 'groups': groups,
         'act': act}
    if op == 'gn_int8':
        c['cout'] = cout
    return dict(c, name=name) if name else c


def _int8(name, dtype, rows, k, n, act):
    c = {'op': 'int8', 'dtype': dtype, 'rows': rows, 'k': k, 'n': n, 'act': act}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one image at 640x640, the stride-32 map of the small model: what a single detection waits for
        _gn('gn', 'gn-one-image', 'fp16', 1, 20, 20, 512, 32, 'leaky'),
        # the stride-4 maps of a serving batch
        _gn('gn', 'gn-batch', 'fp16', 32, 160, 160, 64, 32, 'silu'),
        # a pruned width in a letterboxed batch: odd channel count, odd map
        _gn('gn', 'gn-pruned', 'bf16', 3, 45, 27, 75, 5, 'leaky'),
        # fine-tuning with few images a step, where batch statistics are too noisy
        _gn('gn_train', 'gn-train-few', 'fp32', 4, 40, 40, 256, 32, 'leaky'),
        # a training batch on the stride-8 maps
        _gn('gn_train', 'gn-train-batch', 'bf16', 32, 80, 80, 256, 32, 'silu'),
        # a single token through a square layer
        _int8('int8-token', 'bf16', 1, 4096, 4096, 'none'),
        # few rows into the 255 outputs of a detection head, ragged on every side
        _int8('int8-head-ragged', 'fp16', 333, 1000, 255, 'none'),
        # 1x1 convolution of a serving batch on the stride-32 maps (32 images of 20x20 pixels)
        _int8('int8-deep', 'fp16', 12800, 1024, 512, 'leaky'),
        # 1x1 convolution on the stride-4 maps: narrow, as many pixels as there are
        _int8('int8-narrow', 'fp16', 819200, 64, 64, 'leaky'),
        # a long prompt through a square layer
        _int8('int8-wide', 'bf16', 16384, 4096, 4096, 'none'),
        # norm -> activation -> 1x1 convolution for one image
        _gn('gn_int8', 'gn-int8-one-image', 'fp16', 1, 20, 20, 512, 32, 'leaky', 512),
        # the same for a batch on the stride-8 maps
        _gn('gn_int8', 'gn-int8-batch', 'fp16', 32, 80, 80, 256, 32, 'silu', 256),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(('gn', 'gn_train', 'int8', 'int8', 'gn_int8'))
    # 8-bit layers behind a norm serve 16-bit models: what the rounding of fp32 leaves of a normalised value decides which
    # whole number it becomes, so an fp32 map has nothing to gain there
    dtype = rng.choice(('fp16', 'bf16') if op == 'gn_int8' else ('fp16', 'bf16', 'fp32'))
    act = rng.choice(('none', 'leaky', 'silu'))
    if op == 'int8':
        k, n = _log(rng, 16, 4096), _log(rng, 8, 4096)
        if rng.random() < 0.5:
            k, n = max(16, k // 32 * 32), max(8, n // 32 * 32)
        most = min(819200, int(2e11 / (2.0 * k * n)), 52428800 // max(k, n))
        rows = rng.randint(1, 16) if rng.random() < 0.3 else _log(rng, 1, max(1, most))
        return _int8(None, dtype, rows, k, n, act)
    while True:
        if rng.random() < 0.7:
            groups = rng.choice((8, 16, 32))
            channels = groups * rng.choice((1, 2, 4, 5, 8, 10, 16, 20))
        else:
            groups = rng.randint(1, 12)
            channels = groups * rng.randint(1, 24)
        batch, height, width = _log(rng, 1, 32), _log(rng, 1, 160), _log(rng, 1, 160)
        values = batch * height * width * channels
        # a group of 32 values at least: statistics of fewer say nothing about a map
        if height * width * (channels // groups) >= 32 and 1024 <= values <= 26214400 // (1 if op == 'gn' else 2):
            break
    return _gn(op, None, dtype, batch, height, width, channels, groups, act, _log(rng, 8, 512))


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    t = TYPES[case['dtype']]

    def normal(*shape):
        return torch.randn(shape, generator=g, device='cuda')

    s = dict(case)
    if case['op'] == 'int8':
        # activations with a spread of magnitudes over the rows, as a network's tokens have
        s['x'] = (normal(case['rows'], case['k']) * (0.3 * normal(case['rows'], 1)).exp()).to(t)
        k, n = case['k'], case['n']
    else:
        b, h, w, c = case['batch'], case['height'], case['width'], case['channels']
        # a convolution's raw output: every channel has a mean and a spread of its own
        x = normal(b, h, w, c) * (0.5 * normal(c)).exp() + 0.5 * normal(c)
        s['x'] = x.to(t).permute(0, 3, 1, 2)
        # a half model holds its parameters in half; a training step has fp32 parameters beside 16-bit activations
        p = torch.float32 if case['op'] == 'gn_train' else t
        s['weight'], s['bias'] = (1 + 0.2 * normal(c)).to(p), (0.2 * normal(c)).to(p)
        if case['op'] == 'gn_train':
            s['dy'] = normal(b, h, w, c).to(t).permute(0, 3, 1, 2)
            for name in ('x', 'weight', 'bias'):
                s[name].requires_grad_()
            return s
        k, n = c, case.get('cout', 0)
    if n:
        # the layer as its user keeps it: 8-bit weights with a scale an output channel, fp32 bias
        wf = normal(n, k) * k ** -0.5
        s['wscale'] = wf.abs().amax(1) / 127
        s['wq'] = (wf / s['wscale'][:, None]).round().to(torch.int8)
        s['cbias'] = 0.1 * normal(n)
        if own:
            from yolo_amd import int8
            s['layer'] = int8.Int8Weight(s['wq'], s['wscale'])
    return s


# ---------------------------------------------------------------------------------------------- plain forms

def _act(z, act):
    if act == 'leaky':
        return torch.where(z > 0, z, z * SLOPE)
    if act == 'silu':
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == 'leaky':
        return torch.where(z > 0, 1.0, SLOPE)
    if act == 'silu':
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _normalised(s, x):
    """(normalised values, 1 / standard deviation), as (batch, pixels, groups, channels of a group) and (batch, 1, groups, 1)."""
    b, c = x.shape[:2]
    v = x.permute(0, 2, 3, 1).reshape(b, -1, s['groups'], c // s['groups']).float()
    centred = v - v.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean((1, 3), keepdim=True) + EPS)
    return centred * rstd, rstd


def _map(v, x):
    """(batch, pixels, channels) -> the layout of x."""
    b, c, h, w = x.shape
    return v.reshape(b, h, w, -1).permute(0, 3, 1, 2)


def _plain_rows(x, t):
    """(whole numbers in fp32, scale in fp32) of each row, computed in type t: fp32 results need 64 bits here, because of the
    values next to a half; for 16-bit results 32 do."""
    x = x.to(t)
    a = x.abs().amax(1, keepdim=True)
    some = a >= ZERO_ROW
    q = torch.where(some, x * (127 / torch.where(some, a, 1.0)), 0.0).round()
    return q.float(), torch.where(some, a / 127, 0.0).float()


def _plain_product(q, scale, s, act, dtype):
    # sums of whole numbers below 2^24 are exact in fp32
    y = (q @ s['wq'].float().t()) * (scale * s['wscale']) + s['cbias']
    return _act(y, act).to(dtype)


def _plain(s):
    op, act, x = s['op'], s['act'], s['x'].detach()
    if op == 'int8':
        return _plain_product(*_plain_rows(x, torch.float64 if x.dtype is torch.float32 else torch.float32), s, act, x.dtype)
    b, c, h, w = x.shape
    xhat, rstd = _normalised(s, x)
    shape = (s['groups'], c // s['groups'])
    gamma, beta = s['weight'].detach().float().reshape(shape), s['bias'].detach().float().reshape(shape)
    z = xhat * gamma + beta
    y = _act(z, act)
    if op == 'gn_int8':
        q, scale = _plain_rows(y.reshape(-1, c), torch.float32)
        return _map(_plain_product(q, scale, s, 'none', x.dtype).reshape(b, h * w, -1), x)
    out = _map(y.to(x.dtype), x)
    if op == 'gn':
        return out
    dz = s['dy'].permute(0, 2, 3, 1).reshape(xhat.shape).float() * _act_grad(z, act)
    t = dz * gamma
    dx = rstd * (t - t.mean((1, 3), keepdim=True) - xhat * (t * xhat).mean((1, 3), keepdim=True))
    return {'y': out, 'dx': _map(dx.to(x.dtype), x), 'dgamma': (dz * xhat).sum((0, 1)).reshape(c), 'dbeta': dz.sum((0, 1)).reshape(c)}


def _framework(s):
    from yolo_amd import groupnorm, int8
    op, act, x = s['op'], None if s['act'] == 'none' else s['act'], s['x']
    if op == 'int8':
        return int8.linear_i8(x, s['layer'], s['cbias'], act=act, slope=SLOPE)
    if op == 'gn_int8':
        rows = groupnorm.group_norm_rows(x, s['groups'], s['weight'], s['bias'], EPS, act=act, slope=SLOPE)
        return int8.conv1x1_i8(rows, s['layer'], s['cbias'], dtype=x.dtype)
    y = groupnorm.group_norm(x, s['groups'], s['weight'], s['bias'], EPS, act=act, slope=SLOPE)
    if op == 'gn':
        return y
    dx, dgamma, dbeta = torch.autograd.grad(y, (x, s['weight'], s['bias']), s['dy'])
    return {'y': y, 'dx': dx, 'dgamma': dgamma, 'dbeta': dbeta}


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------- what it has to do

def work(case):
    e = SIZE[case['dtype']]
    if case['op'] == 'int8':
        m, k, n = case['rows'], case['k'], case['n']
        return {'bytes': m * k * e + n * k + 8 * n + m * n * e, 'flops': 2.0 * m * n * k}
    c = case['channels']
    pixels = case['batch'] * case['height'] * case['width']
    if case['op'] == 'gn_int8':
        n = case['cout']
        return {'bytes': pixels * (c + n) * e + n * c + 8 * n + 2 * c * e, 'flops': pixels * c * (2.0 * n + 14)}
    if case['op'] == 'gn_train':
        return {'bytes': 4 * pixels * c * e + 16 * c, 'flops': 32.0 * pixels * c}
    return {'bytes': 2 * pixels * c * e + 2 * c * e, 'flops': 12.0 * pixels * c}


# ---------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    """From the definitions in 64 bits: channel-first, over one axis of all values of a group, with tensor contractions."""
    s = prepare(case, seed)
    with torch.no_grad():
        x = s['x'].detach().double()
        if case['op'] == 'int8':
            return _exact_product(x, s, case['act'])
        b, c, h, w = x.shape
        groups = case['groups']
        v = x.reshape(b, groups, -1)
        n = v.shape[2]
        var, mean = torch.var_mean(v, 2, unbiased=False, keepdim=True)
        sd = (var + EPS).sqrt()
        xhat = ((v - mean) / sd).reshape(b, c, h * w)
        gamma, beta = (s[k].detach().double().reshape(1, c, 1) for k in ('weight', 'bias'))
        z = beta + gamma * xhat
        p = torch.sigmoid(z)
        y = {'none': z, 'leaky': z.clamp(min=0) + SLOPE * z.clamp(max=0), 'silu': z * p}[case['act']]
        if case['op'] == 'gn_int8':
            out = _exact_product(y.transpose(1, 2).reshape(-1, c), s, 'none')
            return out.reshape(b, h, w, -1).permute(0, 3, 1, 2)
        y = y.reshape(b, c, h, w)
        if case['op'] == 'gn':
            return y
        slope = {'none': torch.ones_like(z), 'leaky': SLOPE + (1 - SLOPE) * (z > 0), 'silu': p + z * p * (1 - p)}[case['act']]
        dz = s['dy'].double().reshape(b, c, h * w) * slope
        dxhat = (gamma * dz).reshape(b, groups, n)
        u = xhat.reshape(b, groups, n)
        dx = (n * dxhat - dxhat.sum(2, keepdim=True) - u * (dxhat * u).sum(2, keepdim=True)) / (n * sd)
        return {'y': y, 'dx': dx.reshape(b, c, h, w), 'dgamma': (dz * xhat).sum((0, 2)), 'dbeta': dz.sum((0, 2))}


def _exact_product(x, s, act):
    top = x.abs().amax(1, keepdim=True)
    some = top >= ZERO_ROW
    scale = torch.where(some, top / 127, 0.0)
    q = torch.where(some, x / torch.where(some, scale, 1.0), 0.0).round()
    y = torch.addmm(s['cbias'].double(), q * scale, (s['wq'].double() * s['wscale'].double()[:, None]).t().contiguous())
    return {'none': y, 'leaky': torch.maximum(y, SLOPE * y), 'silu': y * torch.sigmoid(y)}[act]
