"""Cases, plain forms and work of three operators of the channels-last path, as they are measured on a GPU:

  groupnorm    leaky_s(group_norm(x)) on an NHWC tensor, alone or with its backward pass
  linear       leaky_s(x W^T + b) + residual, alone or with its backward pass
  checkpoint   an activation written in 8 bits and read back

`checkpoint8` in the first two: what the backward pass keeps of x is its 8-bit form, so the backward is computed from
that.  A value's 8-bit form: blocks of 32 channels share one power of two 2^e, the smallest with max|x| <= 127 * 2^e,
and a value stands as round(x / 2^e) * 2^e.

With `own` false, run() computes them from elementary torch operations in float32 (float64 where the text says why);
with `own` true it makes the calls of sg2im_amd that a user makes.  Sizes: the refinement network's maps and channels,
the graph convolution's rows and widths, and pixels as rows of a per-pixel perceptron.
"""
import math

import torch

own = False

EPS = 1e-5
BLOCK = 32
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16}


def listed():
  return [
    # the first refinement module's map at batch 32, evaluation: a call of a few microseconds, latency counts
    {'name': 'groupnorm_fwd_f32_4x4', 'op': 'groupnorm', 'train': False, 'type': 'f32', 'n': 32, 'h': 4, 'w': 4, 'c': 1024,
     'groups': 32, 'slope': 0.2, 'checkpoint8': False},
    # the last module's map at 64 x 64, bfloat16 evaluation
    {'name': 'groupnorm_fwd_bf16_64x64', 'op': 'groupnorm', 'train': False, 'type': 'bf16', 'n': 32, 'h': 64, 'w': 64,
     'c': 64, 'groups': 32, 'slope': 0.2, 'checkpoint8': False},
    # the module before it, a float32 training step
    {'name': 'groupnorm_train_f32_32x32', 'op': 'groupnorm', 'train': True, 'type': 'f32', 'n': 32, 'h': 32, 'w': 32,
     'c': 128, 'groups': 32, 'slope': 0.2, 'checkpoint8': False},
    # the last module's map at 256 x 256, bfloat16 training with 8-bit checkpoints: the largest tensor of the framework
    {'name': 'groupnorm_train_bf16_256x256', 'op': 'groupnorm', 'train': True, 'type': 'bf16', 'n': 32, 'h': 256, 'w': 256,
     'c': 64, 'groups': 32, 'slope': 0.2, 'checkpoint8': True},
    # the last linear layer of a graph convolution over one batch's objects, with its residual: latency counts
    {'name': 'linear_fwd_f32_objects', 'op': 'linear', 'train': False, 'type': 'f32', 'm': 203, 'k': 512, 'n': 128,
     'slope': 0.0, 'residual': True, 'checkpoint8': False},
    # a per-pixel perceptron's wide layer over the 32 x 32 map of a batch, evaluation: the largest product
    {'name': 'linear_fwd_bf16_wide', 'op': 'linear', 'train': False, 'type': 'bf16', 'm': 32768, 'k': 1024, 'n': 4096,
     'slope': 0.2, 'residual': False, 'checkpoint8': False},
    # the per-pixel perceptron's second layer at 32 x 32, training, residual, no activation
    {'name': 'linear_train_bf16_pixels', 'op': 'linear', 'train': True, 'type': 'bf16', 'm': 32768, 'k': 1024, 'n': 256,
     'slope': 1.0, 'residual': True, 'checkpoint8': False},
    # its first layer at 64 x 64, training with 8-bit checkpoints: many rows, few channels
    {'name': 'linear_train_bf16_rows8', 'op': 'linear', 'train': True, 'type': 'bf16', 'm': 131072, 'k': 64, 'n': 256,
     'slope': 0.2, 'residual': False, 'checkpoint8': True},
    # the widest linear layer of a graph convolution over the triples of a 256 x 256 batch, float32 training
    {'name': 'linear_train_f32_triples', 'op': 'linear', 'train': True, 'type': 'f32', 'm': 3200, 'k': 512, 'n': 1152,
     'slope': 1.0, 'residual': True, 'checkpoint8': False},
    # widths that no vector load divides (161: the layout's channels next to the seed's), 8-bit checkpoints
    {'name': 'linear_train_bf16_odd8', 'op': 'linear', 'train': True, 'type': 'bf16', 'm': 4099, 'k': 161, 'n': 515,
     'slope': 0.2, 'residual': True, 'checkpoint8': True},
    # the hidden activations of the objects' perceptron, to 8 bits and back
    {'name': 'checkpoint_f32_objects', 'op': 'checkpoint', 'type': 'f32', 'm': 203, 'c': 512},
    # the last module's map at 256 x 256
    {'name': 'checkpoint_bf16_256x256', 'op': 'checkpoint', 'type': 'bf16', 'm': 2097152, 'c': 64},
  ]


def _log(rng, lo, hi):
  return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
  """one more case: every size spread over its range, odd ones among them; never dearer than the largest listed one"""
  op = rng.choice(['groupnorm', 'groupnorm', 'linear', 'linear', 'linear', 'checkpoint'])
  ty = rng.choice(['f32', 'bf16'])
  if op == 'groupnorm':
    groups = rng.choice([1, 2, 4, 8, 16, 20, 32, 32])
    c = groups * _log(rng, 1, 1024 // groups)
    n, h, w = _log(rng, 1, 64), _log(rng, 1, 256), _log(rng, 1, 256)
    cap = (1 << 26) if ty == 'f32' else (1 << 27)
    while n * h * w * c > cap:
      n, h, w = max(1, n // 2), max(1, (h * 2) // 3), max(1, (w * 2) // 3)
    # (a group of one or two values is a constant once it is normalised, and its gradient a difference of equals)
    while h * w * (c // groups) < 16:
      h, w = h + 1, w + 1
    train = rng.random() < 0.6
    return {'op': op, 'train': train, 'type': ty, 'n': n, 'h': h, 'w': w, 'c': c, 'groups': groups,
            'slope': rng.choice([0.0, 0.01, 0.2, 1.0]), 'checkpoint8': train and rng.random() < 0.5}
  if op == 'linear':
    m, k, n = _log(rng, 1, 131072), _log(rng, 16, 4096), _log(rng, 16, 4096)
    if rng.random() < 0.5:
      k, n = -(-k // 8) * 8, -(-n // 8) * 8
    train = rng.random() < 0.6
    # (float32 products run at a sixteenth of bfloat16's rate)
    cap = (1.2e11 if ty == 'bf16' else 1.0e10) / (3 if train else 1)
    while float(m) * k * n > cap or m * max(k, n) > (1 << 27):
      m = max(1, m // 2)
    # Training through a kink: two sums that differ in their last bit fall on different sides of it for a handful of values in
    # a large product, and a float32 gradient is held far closer than that; bfloat16's is not, from some 256 columns on.
    slope = rng.choice([0.0, 0.01, 0.2, 1.0]) if not train or (ty == 'bf16' and n >= 256) else 1.0
    return {'op': op, 'train': train, 'type': ty, 'm': m, 'k': k, 'n': n, 'slope': slope, 'residual': rng.random() < 0.5,
            'checkpoint8': train and rng.random() < 0.4}
  m, c = _log(rng, 1, 2097152), _log(rng, 1, 4096)
  while m * c > (1 << 26):
    m = max(1, m // 2)
  return {'op': op, 'type': ty, 'm': m, 'c': c}


def prepare(case, seed):
  g = torch.Generator(device='cuda')
  g.manual_seed(int(seed))
  ty = TYPES[case['type']]

  def normal(*shape):
    return torch.randn(*shape, device='cuda', dtype=torch.float32, generator=g)

  s = {'case': dict(case)}
  train = case.get('train', False)
  if case['op'] == 'groupnorm':
    n, h, w, c = case['n'], case['h'], case['w'], case['c']
    # what a convolution puts out: every channel has its own mean and spread
    s['x'] = (normal(n, h, w, c) * (0.5 + torch.rand(c, device='cuda', generator=g)) + normal(c)).to(ty)
    s['weight'], s['bias'] = (1 + 0.1 * normal(c)).to(ty), (0.1 * normal(c)).to(ty)
    leaves = ('x', 'weight', 'bias')
    if train:
      s['dy'] = (normal(n, h, w, c) * 0.01).to(ty)
  elif case['op'] == 'linear':
    m, k, n = case['m'], case['k'], case['n']
    s['x'] = normal(m, k).to(ty)
    s['weight'] = (normal(n, k) * math.sqrt(2.0 / k)).to(ty)
    s['bias'] = (0.1 * normal(n)).to(ty)
    s['residual'] = normal(m, n).to(ty) if case['residual'] else None
    leaves = ('x', 'weight', 'bias', 'residual')
    if train:
      s['dy'] = (normal(m, n) * 0.01).to(ty)
  else:
    m, c = case['m'], case['c']
    # what leaves an activation: most of it small, a few large channels
    s['x'] = (normal(m, c) * torch.exp(normal(c))).to(ty)
    leaves = ()
  if train:
    for name in leaves:
      if s[name] is not None:
        s[name].requires_grad_(True)
  return s


# ---- the plain forms ----------------------------------------------------------------------------------------------

def _two_to(e):
  """2^e as float32, exactly: the exponent's bits"""
  return ((e + 127) << 23).view(torch.float32)


def _eight(x):
  """what x's 8-bit form stands for, in float32; every step is exact but the rounding to a whole number"""
  c = x.size(-1)
  pad = -c % BLOCK
  v = x.float()
  if pad:
    v = torch.cat([v, v.new_zeros(v.shape[:-1] + (pad,))], -1)
  v = v.reshape(x.shape[:-1] + ((c + pad) // BLOCK, BLOCK))
  m, k = torch.frexp(v.abs().amax(-1, keepdim=True))           # amax = m * 2^k, 0.5 <= m < 1
  e = torch.where(m <= 127.0 / 128.0, k - 7, k - 6)
  e = torch.where(m == 0, torch.full_like(e, -126), e).clamp(-126, 121)
  q = torch.round(v * _two_to(-e)).clamp(-127, 127)
  return (q * _two_to(e)).reshape(x.shape[:-1] + (c + pad,))[..., :c]


def _groupnorm_plain(s):
  c = s['case']
  n, p, ch, g = c['n'], c['h'] * c['w'], c['c'], c['groups']
  d, slope = ch // g, c['slope']
  x = s['x'].float().view(n, p, g, d)
  weight, bias = s['weight'].float().view(g, d), s['bias'].float().view(g, d)
  # (a group of a 256 x 256 map is a sum of 131 072 values: the statistics are summed in 64 bits)
  mean = x.mean((1, 3), keepdim=True, dtype=torch.float64)
  xc = x - mean.float()
  rstd = (xc.square().mean((1, 3), keepdim=True, dtype=torch.float64) + EPS).rsqrt()
  z = xc * rstd.float() * weight + bias
  y = torch.where(z > 0, z, z * slope).to(s['x'].dtype).view(s['x'].shape)
  if not c['train']:
    return {'y': y}
  dy = s['dy'].float().view(n, p, g, d)
  if c['checkpoint8']:
    xc = _eight(s['x']).view(n, p, g, d) - mean.float()
  xh = xc * rstd.float()
  if slope != 1.0:
    # the slope steps at zero, so the side that a value is on is decided in 64 bits
    xs = (_eight(s['x']) if c['checkpoint8'] else s['x']).double().view(n, p, g, d)
    z64 = xs.mul_(rstd * weight.double()).add_(bias.double() - mean * rstd * weight.double())
    dz = torch.where(z64 > 0, dy, dy * slope)
  else:
    dz = dy
  dbias = dz.sum((0, 1)).view(ch)
  dweight = (dz * xh).sum((0, 1)).view(ch)
  gz = dz * weight
  m1 = gz.mean((1, 3), keepdim=True)
  m2 = (gz * xh).mean((1, 3), keepdim=True)
  dx = (rstd.float() * (gz - m1 - xh * m2)).to(s['x'].dtype).view(s['x'].shape)
  ty = s['x'].dtype
  return {'y': y, 'dx': dx, 'dweight': dweight.to(ty), 'dbias': dbias.to(ty)}


def _linear_plain(s):
  c, x = s['case'], s['x']
  slope, ty = c['slope'], x.dtype
  xf, wf = x.float(), s['weight'].float()
  z = xf @ wf.t() + s['bias'].float()
  y = torch.where(z > 0, z, z * slope)
  if s['residual'] is not None:
    y = y + s['residual'].float()
  y = y.to(ty)
  if not c['train']:
    return {'y': y}
  dy = s['dy'].float()
  dz = torch.where(z > 0, dy, dy * slope)
  if c['checkpoint8']:
    xf = _eight(x)
  out = {'y': y, 'dx': (dz @ wf).to(ty), 'dweight': (dz.t() @ xf).to(ty), 'dbias': dz.sum(0).to(ty)}
  if s['residual'] is not None:
    out['dresidual'] = s['dy']
  return out


# ---- the framework's calls ----------------------------------------------------------------------------------------

def _groupnorm_own(s):
  from sg2im_amd import functional as HF
  c = s['case']
  y = HF.GroupNormAct.apply(s['x'], s['weight'], s['bias'], c['groups'], c['slope'], EPS, c['checkpoint8'])
  if not c['train']:
    return {'y': y}
  dx, dweight, dbias = torch.autograd.grad(y, (s['x'], s['weight'], s['bias']), s['dy'])
  return {'y': y.detach(), 'dx': dx, 'dweight': dweight, 'dbias': dbias}


def _linear_own(s):
  from sg2im_amd import functional as HF
  c = s['case']
  y = HF.LinearResidual.apply(s['x'], s['weight'], s['bias'], s['residual'], c['slope'], c['checkpoint8'])
  if not c['train']:
    return {'y': y}
  leaves = [s['x'], s['weight'], s['bias']] + ([s['residual']] if s['residual'] is not None else [])
  grads = torch.autograd.grad(y, leaves, s['dy'])
  out = {'y': y.detach(), 'dx': grads[0], 'dweight': grads[1], 'dbias': grads[2]}
  if s['residual'] is not None:
    out['dresidual'] = grads[3]
  return out


def _checkpoint_own(s):
  from sg2im_amd import ops
  return {'x8': ops.unpack8(ops.pack8(s['x']))}


def run(state):
  op = state['case']['op']
  if own:
    return {'groupnorm': _groupnorm_own, 'linear': _linear_own, 'checkpoint': _checkpoint_own}[op](state)
  with torch.no_grad():
    if op == 'groupnorm':
      return _groupnorm_plain(state)
    if op == 'linear':
      return _linear_plain(state)
    return {'x8': _eight(state['x']).to(state['x'].dtype)}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _exact_eight(x):
  """the 8-bit form's value of a float64 matrix, from its definition: the smallest 2^e with max <= 127 * 2^e"""
  rows, ch = x.shape
  out = torch.empty_like(x)
  for c0 in range(0, ch, BLOCK):
    b = x[:, c0:c0 + BLOCK]
    top = b.abs().max(1, keepdim=True).values
    e = torch.ceil(torch.log2(top.clamp(min=1e-45) / 127))
    power = lambda k: ((k.long() + 1023) << 52).view(torch.float64)  # noqa: E731
    e = torch.where(top > 127 * power(e), e + 1, e)            # (log2 is rounded: look one step to both sides)
    e = torch.where(top <= 127 * power(e - 1), e - 1, e)
    scale = power(e.clamp(-126, 121))
    out[:, c0:c0 + BLOCK] = (b / scale).round().clamp(-127, 127) * scale
  return out


@torch.no_grad()
def exact(case, seed):
  s = prepare(case, seed)
  f = torch.float64
  if case['op'] == 'checkpoint':
    return {'x8': _exact_eight(s['x'].to(f)).to(torch.float32)}
  if case['op'] == 'linear':
    x, w, b = s['x'].to(f), s['weight'].to(f), s['bias'].to(f)
    z = torch.addmm(b, x, w.t())
    y = torch.nn.functional.leaky_relu(z, case['slope'])
    if s['residual'] is not None:
      y += s['residual'].to(f)
    if not case['train']:
      return {'y': y}
    dz = s['dy'].to(f)
    dz[z <= 0] *= case['slope']
    xs = _exact_eight(x) if case['checkpoint8'] else x
    out = {'y': y, 'dx': torch.mm(dz, w), 'dweight': torch.mm(xs.t(), dz).t().contiguous(), 'dbias': dz.sum(0)}
    if s['residual'] is not None:
      out['dresidual'] = s['dy'].to(f)
    return out
  n, p, ch, g = case['n'], case['h'] * case['w'], case['c'], case['groups']
  y, dx = [], []
  dw, db = torch.zeros(ch, device='cuda', dtype=f), torch.zeros(ch, device='cuda', dtype=f)
  w, b = s['weight'].to(f), s['bias'].to(f)
  for i in range(n):                                           # one image at a time, groups in front
    x = s['x'][i].to(f).view(p, ch)
    rows = x.view(p, g, ch // g).permute(1, 0, 2).reshape(g, -1)
    mean = rows.mean(1).repeat_interleave(ch // g)
    std = torch.sqrt(rows.var(1, unbiased=False) + EPS).repeat_interleave(ch // g)
    z = (x - mean) / std * w + b
    y.append(torch.nn.functional.leaky_relu(z, case['slope']))
    if case['train']:
      xs = _exact_eight(x) if case['checkpoint8'] else x
      hat = (xs - mean) / std
      dz = s['dy'][i].to(f).view(p, ch).clone()
      dz[hat * w + b <= 0] *= case['slope']
      dw += (dz * hat).sum(0)
      db += dz.sum(0)
      t = dz * w
      per = lambda v: v.sum(0).view(g, -1).sum(1).repeat_interleave(ch // g) / (p * (ch // g))  # noqa: E731
      dx.append((t - per(t) - hat * per(t * hat)) / std)
  shape = (n, case['h'], case['w'], ch)
  out = {'y': torch.stack(y).view(shape)}
  if case['train']:
    out.update(dx=torch.stack(dx).view(shape), dweight=dw, dbias=db)
  return out


def work(case):
  """each input read once, each output written once; an 8-bit form is written by the forward and read by the backward pass"""
  es = 4 if case['type'] == 'f32' else 2
  if case['op'] == 'groupnorm':
    e, c = float(case['n'] * case['h'] * case['w'] * case['c']), case['c']
    if not case['train']:
      return {'bytes': 2 * e * es + 2 * es * c, 'flops': 8 * e}
    return {'bytes': 4 * e * es + 4 * es * c + (2 * e * 33 / 32 if case['checkpoint8'] else 0), 'flops': 24 * e}
  if case['op'] == 'linear':
    m, k, n = float(case['m']), case['k'], case['n']
    r = 1 if case['residual'] else 0
    if not case['train']:
      return {'bytes': es * (m * k + n * k + (1 + r) * m * n + n), 'flops': 2 * m * n * k}
    return {'bytes': es * (2 * m * k + 2 * n * k + (2 + r) * m * n + 2 * n) + (2 * m * k * 33 / 32 if case['checkpoint8'] else 0),
            'flops': 6 * m * n * k}
  e = float(case['m'] * case['c'])
  return {'bytes': 2 * e * es + 2 * e * 33 / 32, 'flops': 4 * e}
