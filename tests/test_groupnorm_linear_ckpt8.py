"""Group norm + activation, linear + activation + residual and 8-bit activation checkpoints against their definitions in 64
bits.  Tolerances are bounds of the arithmetic, element by element, with u = 2^-24 (half a step of float32) and U = half a
step of the output's type (eps / 2):

  group norm  z = fma(x - m, a, b): three roundings of the product's side, one of b, one of z, one of the slope
  sums        a thread adds at most T values in float32 before they are joined in 64 bits: T u of the absolute sum
  linear      any order of K products in float32: K u of the absolute sum, then bias, slope and residual
"""
import ctypes
import itertools
import math

import pytest
import torch

gpu = pytest.mark.gpu
F64, F32, BF16 = torch.float64, torch.float32, torch.bfloat16
u32 = 2.0 ** -24
T = 16          # float32 additions in a row per thread, at the sizes of this file


def half_step(dtype):
  return torch.finfo(dtype).eps / 2


def check(got, want, tol, what):
  got, want = got.detach().to(F64), want.to(F64)
  assert got.shape == want.shape, (what, got.shape, want.shape)
  bad = ~((got - want).abs() <= tol) & ~(got.isnan() & want.isnan()) & ~(got == want)
  if bool(bad.any()):
    k = int(bad.flatten().nonzero()[0])
    raise AssertionError('%s: %d of %d out of bounds, first at %d: %r, want %r +- %r'
                         % (what, int(bad.sum()), bad.numel(), k, float(got.flatten()[k]), float(want.flatten()[k]),
                            float(tol.expand_as(want).flatten()[k]) if torch.is_tensor(tol) else tol))


def gen(seed):
  g = torch.Generator(device='cuda')
  g.manual_seed(seed)
  return lambda *s: torch.randn(*s, device='cuda', generator=g)


# ---- the 8-bit form -------------------------------------------------------------------------------------------------

def eight(x):
  """the 8-bit form's values in float64 and their exponents, from the definition; what is not finite becomes NaN"""
  C = x.size(-1)
  v = x.to(F64).reshape(-1, C)
  out, exps = torch.empty_like(v), []
  for c0 in range(0, C, 32):
    b = v[:, c0:c0 + 32]
    fin = torch.isfinite(b)
    m, k = torch.frexp(torch.where(fin, b, torch.zeros_like(b)).abs().amax(1, keepdim=True))
    e = torch.where(m <= 127.0 / 128.0, k - 7, k - 6)
    e = torch.where(m == 0, torch.full_like(e, -126), e).clamp(-126, 121)
    scale = torch.pow(torch.tensor(2.0, dtype=F64), e.cpu().to(F64)).to(v.device)
    q = torch.where(fin, torch.round(torch.where(fin, b, torch.zeros_like(b)) / scale).clamp(-127, 127),
                    torch.full_like(b, math.nan))
    out[:, c0:c0 + 32] = q * scale
    exps.append(e + 127)
  return out.reshape(x.shape), torch.cat(exps, 1).to(torch.uint8).reshape(x.shape[:-1] + (len(exps),))


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('shape', [(1, 1), (3, 31), (5, 32), (7, 33), (203, 512), (64, 161), (2, 3, 5, 64), (0, 40), (9, 4099)])
def test_pack8_is_the_definition(shape, dtype):
  from sg2im_amd import ops
  r = gen(1)
  x = (r(*shape) * torch.exp(4 * r(shape[-1]))).to(dtype)
  p = ops.pack8(x)
  want, exps = eight(x)
  got = ops.unpack8(p)
  assert got.dtype == dtype and got.shape == x.shape
  assert torch.equal(got.to(F64), want) and torch.equal(p.exps, exps)
  assert torch.equal(ops.unpack8(p, F32).to(F64), want) and torch.equal(ops.unpack8(p, BF16).to(F64), want)


@gpu
def test_pack8_extremes_and_strides():
  from sg2im_amd import ops
  big = torch.finfo(F32).max
  rows = [[0.0] * 32, [1e-45] + [0.0] * 31, [big] * 32, [-big, 1.0] + [0.0] * 30, [math.inf, 1.0, -2.0] + [0.5] * 29,
          [math.nan] * 32, [-math.inf, 127.0] + [0.25] * 30, [127.0 * 2.0 ** k for k in range(-16, 16)],
          [127.5] + [0.5, 1.5, 2.5, -0.5, -1.5] + [0.0] * 26, [2.0 ** -130] * 32]
  x = torch.tensor(rows, device='cuda')
  for t in (x, x.to(BF16)):
    got, (want, exps) = ops.unpack8(ops.pack8(t)), eight(t)
    assert torch.equal(got.to(F64).nan_to_num(nan=12345.0), want.nan_to_num(nan=12345.0))
    assert torch.equal(ops.pack8(t).exps, exps)
  wide = gen(2)(50, 301).to(BF16)
  for view in (wide[:, 7:170], wide[::3, 1:34], wide.t()[:, :40], wide[:1, 5:6].expand(6, 1)):
    assert torch.equal(ops.unpack8(ops.pack8(view)).to(F64), eight(view)[0])
  # the error is at most half a step of the block
  t = gen(3)(100, 96)
  got, exps = ops.unpack8(ops.pack8(t)), eight(t)[1]
  step = torch.pow(2.0, exps.to(F64) - 127).repeat_interleave(32, 1)
  assert bool(((got - t).abs().to(F64) <= step / 2).all())


# ---- group norm -----------------------------------------------------------------------------------------------------

def gn_reference(x, xs, w, b, groups, slope, eps, dy):
  """values and absolute sums of the formula in 64 bits; xs: what the backward pass sees of x"""
  shape, C = x.shape, x.size(-1)
  N, D = shape[0], C // groups
  v = lambda t: t.to(F64).reshape(N, -1, groups, D)  # noqa: E731
  w = (w.to(F64) if w is not None else torch.ones(C, device=x.device, dtype=F64)).view(groups, D)
  b = (b.to(F64) if b is not None else torch.zeros(C, device=x.device, dtype=F64)).view(groups, D)
  x, xs = v(x), v(xs)
  mean = x.mean((1, 3), keepdim=True)
  rstd = ((x - mean).square().mean((1, 3), keepdim=True) + eps).rsqrt()
  xh = (x - mean) * rstd
  z = xh * w + b
  y = torch.where(z > 0, z, z * slope)
  r = {'y': y.reshape(shape), 'y_tol': (6 * u32 * ((xh * w).abs() + b.abs())).reshape(shape)}
  if dy is None:
    return r
  xh = (xs - mean) * rstd
  dz = v(dy) * torch.where(xh * w + b > 0, 1.0, float(slope))
  gz, A = dz * w, lambda t: t.abs().mean((1, 3), keepdim=True)  # noqa: E731
  m1, m2 = gz.mean((1, 3), keepdim=True), (gz * xh).mean((1, 3), keepdim=True)
  r['dx'] = (rstd * (gz - m1 - xh * m2)).reshape(shape)
  r['dx_tol'] = (rstd * u32 * (5 * gz.abs() + (T + 5) * A(gz) + xh.abs() * (T + 10) * A(gz * xh))).reshape(shape)
  r['dw'], r['dw_tol'] = (dz * xh).sum((0, 1)).reshape(-1), (T + 8) * u32 * (dz * xh).abs().sum((0, 1)).reshape(-1)
  r['db'], r['db_tol'] = dz.sum((0, 1)).reshape(-1), (T + 4) * u32 * dz.abs().sum((0, 1)).reshape(-1)
  return r


GN_SHAPES = [((1, 1, 1, 8), 1), ((2, 4, 4, 1024), 32), ((3, 5, 7, 48), 3), ((2, 9, 11, 105), 5), ((1, 64, 64, 64), 32),
             ((5, 1, 1, 32), 2), ((2, 3, 3, 7), 7), ((1, 13, 1, 2100), 4), ((4, 6, 5, 1), 1), ((70, 2, 2, 64), 8),
             ((1, 1, 1, 33), 1), ((2, 31, 33, 160), 20), ((1, 200, 3, 30), 1)]
GN_TYPES = [(F32, F32, F32), (BF16, BF16, BF16), (BF16, BF16, F32), (F32, BF16, F32)]     # x, y, parameters


@gpu
@pytest.mark.parametrize('types', GN_TYPES)
@pytest.mark.parametrize('shape,groups', GN_SHAPES)
def test_group_norm_forward_and_backward(shape, groups, types):
  from sg2im_amd import functional as HF
  tx, ty, tp = types
  r = gen(hash((shape, groups)) % 1000)
  C = shape[-1]
  x0 = (r(*shape) * (0.5 + r(C).abs()) + r(C)).to(tx)
  w0, b0 = (1 + 0.2 * r(C)).to(tp), (0.2 * r(C)).to(tp)
  dy = r(*shape).to(ty)
  for slope, ckpt in ((0.2, False), (1.0, True), (0.0, True), (0.01, False)):
    x, w, b = (t.clone().requires_grad_(True) for t in (x0, w0, b0))
    y = HF.GroupNormAct.apply(x, w, b, groups, slope, 1e-5, ckpt, ty)
    assert y.dtype == ty
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert (dx.dtype, dw.dtype, db.dtype) == (tx, tp, tp)
    ref = gn_reference(x0, eight(x0)[0] if ckpt else x0, w0, b0, groups, slope, 1e-5, dy)
    check(y, ref['y'], ref['y_tol'] + half_step(ty) * ref['y'].abs(), 'y')
    check(dx, ref['dx'], ref['dx_tol'] + half_step(tx) * ref['dx'].abs(), 'dx')
    check(dw, ref['dw'], ref['dw_tol'] + half_step(tp) * ref['dw'].abs(), 'dweight')
    check(db, ref['db'], ref['db_tol'] + half_step(tp) * ref['db'].abs(), 'dbias')


@gpu
def test_group_norm_gradient_against_differences():
  """central differences, in 64 bits, of the definition's loss: an answer that does not know the gradient's formula"""
  from sg2im_amd import functional as HF
  r = gen(5)
  x0, w0, b0, dy = r(2, 5, 6, 24), 1 + 0.2 * r(24), 0.2 * r(24), r(2, 5, 6, 24)
  # (0.3 below: z keeps 1e-3 from the kink, a thousand steps of the difference)
  loss = lambda x, w, b: (gn_reference(x, x, w, b, 4, 0.3, 1e-5, None)['y'] * dy.to(F64)).sum()  # noqa: E731
  for _ in range(20):
    z = gn_reference(x0, x0, w0, b0, 4, 1.0, 1e-5, None)['y']
    if float(z.abs().min()) > 1e-3:
      break
    x0 = x0 + 0.05 * (z.abs() <= 1e-3)
  x, w, b = (t.clone().requires_grad_(True) for t in (x0, w0, b0))
  grads = torch.autograd.grad(HF.GroupNormAct.apply(x, w, b, 4, 0.3), (x, w, b), dy)
  ref = gn_reference(x0, x0, w0, b0, 4, 0.3, 1e-5, dy)
  h = 1e-6
  for k, (name, g) in enumerate(zip(('dx', 'dw', 'db'), grads)):
    d = r(*g.shape).to(F64)
    at = lambda s: loss(*[t.to(F64) + (s * h * d if j == k else 0) for j, t in enumerate((x0, w0, b0))])  # noqa: E731,B023
    want = float(at(1) - at(-1)) / (2 * h)
    tol = ((ref[name + '_tol'] + u32 * ref[name].abs()) * d.abs()).sum()
    # (the difference: 2^-53 of the loss' absolute sum over h, and a third derivative of order 1 times h^2)
    tol = float(tol) + 2.0 ** -52 * float(dy.abs().sum()) * 8 / h + 1e-9
    assert abs(float((g.to(F64) * d).sum()) - want) <= tol, name


@gpu
def test_group_norm_far_mean_kink_and_missing_parameters():
  from sg2im_amd import functional as HF
  r = gen(7)
  # a mean of a thousand deviations: 24 bits of x leave 14 for the difference, and no more is lost
  x0 = (1000 + r(2, 16, 16, 32)).requires_grad_(True)
  dy = r(2, 16, 16, 32)
  y = HF.GroupNormAct.apply(x0, None, None, 8, 0.2)
  (dx,) = torch.autograd.grad(y, (x0,), dy)
  ref = gn_reference(x0.detach(), x0.detach(), None, None, 8, 0.2, 1e-5, dy)
  check(y, ref['y'], ref['y_tol'] + u32 * ref['y'].abs(), 'y')
  check(dx, ref['dx'], ref['dx_tol'] + u32 * ref['dx'].abs(), 'dx')
  # values that lie on the kink: x is -1, 0, 1 in equal parts, so z is exactly 0 for a third of them (the slope applies)
  pat = torch.tensor([-1.0, 0.0, 1.0], device='cuda').repeat(32).view(1, 6, 4, 4).clone().requires_grad_(True)
  b = torch.zeros(4, device='cuda', requires_grad=True)
  (db,) = torch.autograd.grad(HF.GroupNormAct.apply(pat, None, b, 2, 0.25), (b,), torch.ones(1, 6, 4, 4, device='cuda'))
  want = torch.where(pat > 0, 1.0, 0.25).sum((0, 1, 2))
  assert torch.equal(db, want)
  # a bias that puts z within a rounding of the kink: decided as in 64 bits
  x = r(1, 64, 64, 2).requires_grad_(True)
  xd = x.detach().to(F64)
  m, s = xd.mean(), xd.var(unbiased=False)
  z0 = ((xd - m) / torch.sqrt(s + 1e-5)).flatten()[777]
  b = torch.full((2,), float((-z0).to(F32)), device='cuda', requires_grad=True)
  y = HF.GroupNormAct.apply(x, None, b, 1, 0.0)
  (db,) = torch.autograd.grad(y, (b,), torch.ones_like(y))
  want = ((xd - m) / torch.sqrt(s + 1e-5) + b.detach().to(F64) > 0).to(F32).sum((0, 1, 2))
  assert torch.equal(db, want)


@gpu
def test_group_norm_not_finite_empty_and_strided():
  from sg2im_amd import functional as HF
  r = gen(8)
  x = r(3, 4, 4, 64)
  clean = HF.GroupNormAct.apply(x, None, None, 4, 0.2)
  x[1, 2, 3, 20] = math.nan
  x[2, 0, 0, 63] = math.inf
  y = HF.GroupNormAct.apply(x, None, None, 4, 0.2)
  assert bool(y[1, :, :, 16:32].isnan().all()) and bool(y[2, :, :, 48:].isnan().all())
  keep = torch.ones_like(y, dtype=torch.bool)
  keep[1, :, :, 16:32] = keep[2, :, :, 48:] = False
  assert torch.equal(y[keep], clean[keep])
  # the gradient of the others stays, from x and from its 8-bit form
  for ckpt in (False, True):
    xs = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(HF.GroupNormAct.apply(xs, None, None, 4, 0.2, 1e-5, ckpt), (xs,), torch.ones_like(x))
    assert bool(dx[1, :, :, 16:32].isnan().all()) and bool(dx[keep].isfinite().all())
  # no image
  e = torch.empty(0, 4, 4, 64, device='cuda', requires_grad=True)
  w = torch.ones(64, device='cuda', requires_grad=True)
  y = HF.GroupNormAct.apply(e, w, None, 4, 0.2, 1e-5, True)
  de, dw = torch.autograd.grad(y, (e, w), torch.empty_like(y))
  assert y.shape == e.shape and de.shape == e.shape and torch.equal(dw, torch.zeros(64, device='cuda'))
  # channels-first memory, an expanded gradient
  nchw = r(2, 32, 5, 7)
  a = nchw.permute(0, 2, 3, 1).requires_grad_(True)
  y = HF.GroupNormAct.apply(a, None, None, 4, 0.2)
  (g1,) = torch.autograd.grad(y.sum(), (a,))
  b = a.detach().contiguous().requires_grad_(True)
  y2 = HF.GroupNormAct.apply(b, None, None, 4, 0.2)
  (g2,) = torch.autograd.grad(y2, (b,), torch.ones_like(y2))
  assert torch.equal(y, y2) and torch.equal(g1, g2)


# ---- linear ---------------------------------------------------------------------------------------------------------

def lin_bounds(x, xs, w, b, res, slope, dy, bits, t_op, dz_type):
  """values and bounds in 64 bits; bits: the sides z > 0 that the forward pass kept"""
  x, xs, w = x.to(F64), xs.to(F64), w.to(F64)
  M, K, N = x.size(0), x.size(1), w.size(0)
  z = x @ w.t() + (b.to(F64) if b is not None else 0)
  az = x.abs() @ w.abs().t() + (b.to(F64).abs() if b is not None else 0)
  r = {'z': z, 'z_tol': (K + 3) * u32 * az}
  y = torch.where(z > 0, z, z * slope)
  r['y'] = y + (res.to(F64) if res is not None else 0)
  r['y_tol'] = r['z_tol'] * max(1.0, abs(slope)) + 2 * u32 * (y.abs() + (res.to(F64).abs() if res is not None else 0))
  dz = dy.to(F64) * (torch.where(bits, 1.0, float(slope)) if bits is not None else 1.0)
  # (dz is rounded to the products' type unless it is dy itself)
  rz = 0.0 if bits is None and dy.dtype == t_op else half_step(t_op)
  r['dx'], r['dx_tol'] = dz @ w, ((N + 2) * u32 + rz) * (dz.abs() @ w.abs())
  r['dw'], r['dw_tol'] = dz.t() @ xs, ((M + 2) * u32 + rz) * (dz.abs().t() @ xs.abs())
  # (a thread adds up four rows of a chunk of 32, then the chunks, then 32 threads, then the splits)
  r['db'], r['db_tol'] = dz.sum(0), (4 + M / 32 + 32 + 128) * u32 * dz.abs().sum(0)
  return r


def sides(words, N):
  k = torch.arange(N, device=words.device)
  return (words[:, k // 32] >> (k % 32) & 1).bool()


LIN_SIZES = [(1, 1, 1), (1, 16, 40), (5, 7, 3), (64, 64, 64), (203, 512, 128), (129, 161, 515), (300, 1024, 256),
             (1000, 96, 1152), (4099, 64, 40), (70, 2600, 33), (3, 4096, 4096), (513, 130, 258), (20000, 33, 17)]


@gpu
@pytest.mark.parametrize('types', [(F32, F32, F32), (BF16, BF16, BF16), (BF16, F32, BF16), (BF16, BF16, F32)])      # x, y, weight
@pytest.mark.parametrize('size', LIN_SIZES)
def test_linear_forward_and_backward(size, types):
  from sg2im_amd import functional as HF, ops
  M, K, N = size
  tx, ty, tw = types
  r = gen(M + K + N)
  x0, w0, b0 = r(M, K).to(tx), (r(N, K) / math.sqrt(K)).to(tw), (0.1 * r(N)).to(tw)
  res0, dy = r(M, N).to(ty), r(M, N).to(ty)
  wx = w0.to(tx)                                          # (a float32 weight next to a bfloat16 x is rounded)
  for slope, ckpt, use_res, use_bias in ((0.2, False, True, True), (1.0, True, False, True), (0.0, True, True, False),
                                         (1.0, False, True, True)):
    x, w, b, res = (t.clone().requires_grad_(True) for t in (x0, w0, b0, res0))
    args = [x, w] + ([b] if use_bias else []) + ([res] if use_res else [])
    y = HF.LinearResidual.apply(x, w, b if use_bias else None, res if use_res else None, slope, ckpt, ty)
    grads = dict(zip(['dx', 'dw'] + (['db'] if use_bias else []) + (['dres'] if use_res else []),
                     torch.autograd.grad(y, args, dy)))
    bits = None
    if slope != 1.0:
      bits = sides(ops.linear_forward(x0, wx, b0 if use_bias else None, None, slope, ty, signs=True)[1], N)
    f = lin_bounds(x0, eight(x0)[0] if ckpt else x0, wx, b0 if use_bias else None, res0 if use_res else None, slope, dy, bits,
                   tx, ty)
    if bits is not None:
      wrong = bits != (f['z'] > 0)
      assert not bool((wrong & (f['z'].abs() > f['z_tol'])).any()), 'sides'
    assert y.dtype == ty and grads['dx'].dtype == tx and grads['dw'].dtype == tw
    check(y, f['y'], f['y_tol'] + half_step(ty) * f['y'].abs(), 'y')
    check(grads['dx'], f['dx'], f['dx_tol'] + half_step(tx) * f['dx'].abs(), 'dx')
    check(grads['dw'], f['dw'], f['dw_tol'] + half_step(tw) * f['dw'].abs(), 'dweight')
    if use_bias:
      check(grads['db'], f['db'], f['db_tol'] + half_step(tw) * f['db'].abs(), 'dbias')
    if use_res:
      assert torch.equal(grads['dres'], dy)


@gpu
@pytest.mark.parametrize('ty', [F32, BF16])
@pytest.mark.parametrize('K', [3, 4, 8, 9, 31, 33, 100, 257, 516, 1100])
def test_small_forward_products(K, ty):
  """few outputs, every remainder of a row's end, strided rows; signs of rows' half words"""
  from sg2im_amd import ops
  for M, N in ((1, 1), (7, 18), (16, 16), (17, 35), (33, 61), (50, 96)):
    r = gen(100 * K + M + N)
    x, w = r(M, K + 5).to(ty)[:, 3:3 + K], (r(N, K) / math.sqrt(K)).to(ty)
    b, res = r(N).to(ty), r(M, N).to(ty)
    y, signs = ops.linear_forward(x, w, b, res, 0.2, ty, signs=True)
    f = lin_bounds(x, x, w, b, res, 0.2, res, sides(signs, N), ty, ty)
    check(y, f['y'], f['y_tol'] + half_step(ty) * f['y'].abs(), 'y')
    wrong = sides(signs, N) != (f['z'] > 0)
    assert not bool((wrong & (f['z'].abs() > f['z_tol'])).any()), 'sides'
    assert signs.shape == (M, (N + 31) // 32)
    if N % 32:
      assert not bool((signs[:, -1].long() & 0xffffffff >> N % 32 << N % 32).any()), 'bits past the last column'


@gpu
def test_linear_gradient_against_differences():
  """the loss is linear in each of x, W, b and the residual away from the kink: a difference of the definition is exact"""
  from sg2im_amd import functional as HF
  r = gen(11)
  x0, w0, b0, res0, dy = r(37, 24), r(19, 24), r(19), r(37, 19), r(37, 19)

  def loss(x, w, b, res):
    z = x @ w.t() + b
    return ((torch.where(z > 0, z, z * 0.3) + res) * dy.to(F64)).sum()
  z = x0.to(F64) @ w0.to(F64).t() + b0.to(F64)
  dy = dy * (z.abs() > 1e-3)                     # (what lies nearer to the kink than the difference's step does not count)
  leaves = [t.clone().requires_grad_(True) for t in (x0, w0, b0, res0)]
  grads = torch.autograd.grad(HF.LinearResidual.apply(*leaves, 0.3), leaves, dy)
  bits = z > 0
  f = lin_bounds(x0, x0, w0, b0, res0, 0.3, dy, bits, F32, F32)
  f['dr'], f['dr_tol'] = dy.to(F64), torch.zeros((), dtype=F64, device='cuda')
  h = 2.0 ** -20
  for k, (name, g) in enumerate(zip(('dx', 'dw', 'db', 'dr'), grads)):
    d = r(*g.shape).to(F64)
    at = lambda s: loss(*[t.to(F64) + (s * h * d if j == k else 0) for j, t in enumerate((x0, w0, b0, res0))])  # noqa: E731,B023
    want = float(at(1) - at(-1)) / (2 * h)
    mag = float(((x0.to(F64).abs() @ w0.to(F64).abs().t() + 4) * dy.to(F64).abs()).sum())
    tol = float(((f[name + '_tol'] + u32 * f[name].abs()) * d.abs()).sum()) + 64 * 2.0 ** -52 * mag / h
    assert abs(float((g.to(F64) * d).sum()) - want) <= tol, name


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_linear_strides_alignment_and_leading_dims(dtype):
  from sg2im_amd import functional as HF
  r = gen(12)
  wide = r(60, 200).to(dtype)
  w, b = (r(48, 72) / 8).to(dtype), r(48).to(dtype)
  dense = lambda t: HF.LinearResidual.apply(t.contiguous(), w, b, None, 0.2)  # noqa: E731
  for x in (wide[:, 3:75], wide[::2, 128:], wide.t()[:72, :].t(), wide[:1, :72].expand(9, 72), wide[5:6, 1:73]):
    assert torch.equal(HF.LinearResidual.apply(x, w, b, None, 0.2), dense(x))
  flat = torch.zeros(60 * 72 + 1, device='cuda', dtype=dtype)
  flat[1:] = wide[:, :72].reshape(-1)
  odd = flat[1:].view(60, 72)                                          # one element off every alignment
  assert torch.equal(HF.LinearResidual.apply(odd, w, b, None, 0.2), dense(odd))
  x4 = wide[:, :72].reshape(3, 4, 5, 72).contiguous().requires_grad_(True)
  res = r(3, 4, 5, 48).to(dtype).permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3)
  y = HF.LinearResidual.apply(x4, w, b, res, 0.2)
  y2 = HF.LinearResidual.apply(x4.detach().reshape(60, 72), w, b, res.reshape(60, 48), 0.2)
  assert y.shape == (3, 4, 5, 48) and torch.equal(y.reshape(60, 48), y2)
  (g,) = torch.autograd.grad(y.sum(), (x4,))
  assert g.shape == x4.shape
  # no row
  e = torch.empty(0, 72, device='cuda', dtype=dtype, requires_grad=True)
  wl, bl = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
  for ckpt in (False, True):
    y = HF.LinearResidual.apply(e, wl, bl, None, 0.2, ckpt)
    de, dw, db = torch.autograd.grad(y, (e, wl, bl), torch.empty_like(y))
    assert y.shape == (0, 48) and de.shape == e.shape and not bool(dw.any()) and not bool(db.any())


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_linear_not_finite_stays_in_its_rows(dtype):
  from sg2im_amd import functional as HF
  r = gen(13)
  x, w = r(100, 72).to(dtype), (r(50, 72) / 8).to(dtype)
  clean = HF.LinearResidual.apply(x, w, None, None, 0.2)
  x[17, 71], x[40, 0] = math.nan, math.inf
  y = HF.LinearResidual.apply(x, w, None, None, 0.2)
  keep = torch.ones(100, dtype=torch.bool, device='cuda')
  keep[17] = keep[40] = False
  assert torch.equal(y[keep], clean[keep]) and bool(y[17].isnan().all()) and not bool(y[40].isfinite().any())


# ---- together -------------------------------------------------------------------------------------------------------

def chain(x, p, ckpt):
  from sg2im_amd import functional as HF
  h = HF.GroupNormAct.apply(x, p['gw'], p['gb'], 8, 0.2, 1e-5, ckpt)
  h = HF.LinearResidual.apply(h, p['w1'], p['b1'], None, 0.2, ckpt)
  return HF.LinearResidual.apply(h, p['w2'], p['b2'], x, 1.0, ckpt)


def chain_params(dtype, C=64, Hd=160):
  r = gen(21)
  p = {'gw': 1 + 0.1 * r(C), 'gb': 0.1 * r(C), 'w1': r(Hd, C) / 8, 'b1': 0.1 * r(Hd), 'w2': r(C, Hd) / 13, 'b2': 0.1 * r(C)}
  return {k: v.to(dtype).requires_grad_(True) for k, v in p.items()}


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('ckpt', [False, True])
def test_the_three_together_on_streams_and_in_graphs(dtype, ckpt):
  """a residual block of group norm and two linear layers: bit-equal on another stream, in two captured graphs replayed with
  eager work between, and next to another call in flight"""
  p = chain_params(dtype)
  r = gen(22)
  x = r(4, 16, 16, 64).to(dtype).requires_grad_(True)
  dy = r(4, 16, 16, 64).to(dtype)
  leaves = [x] + list(p.values())
  run = lambda: torch.autograd.grad(chain(x, p, ckpt), leaves, dy)  # noqa: E731
  want = [chain(x, p, ckpt).detach()] + list(run())
  same = lambda got: all(torch.equal(a, b) for a, b in zip(got, want))  # noqa: E731
  assert same([chain(x, p, ckpt).detach()] + list(run()))
  side = [torch.cuda.Stream() for _ in range(2)]
  outs = []
  for s in side * 2:
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
      outs.append([chain(x, p, ckpt).detach()] + list(run()))
  torch.cuda.synchronize()
  assert all(same(o) for o in outs)
  graphs = []
  for _ in range(2):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      y = chain(x, p, ckpt)
      out = [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    graphs.append((g, out))
  keep = x.detach().clone()
  for k in range(3):
    with torch.no_grad():
      x.copy_(keep if k != 1 else keep * 0.5)
    want = [chain(x, p, ckpt).detach()] + list(run())
    for (g, out), s in zip(graphs, side):
      for o in out:
        o.fill_(7.0)
      s.wait_stream(torch.cuda.current_stream())
      with torch.cuda.stream(s):
        g.replay()
    torch.cuda.synchronize()
    assert all(same(out) for _, out in graphs)
    run()


@gpu
def test_capture_next_to_a_living_graph_of_the_same_leaves_is_refused():
  """the leaf's accumulation node would be one of the default stream; released, or with a sink, the capture goes through"""
  from sg2im_amd import functional as HF
  r = gen(33)
  x, w, b = r(6, 32).requires_grad_(True), r(32, 32).requires_grad_(True), r(32).requires_grad_(True)
  dy = r(6, 32)
  calls = {'group norm': (lambda x, w, b: HF.GroupNormAct.apply(x, b, None, 4, 0.2), (x, b)),
           'linear': (lambda x, w, b: HF.LinearResidual.apply(x, w, b, x, 0.2), (x, w, b))}
  for name, (call, leaves) in calls.items():
    y = call(x, w, b)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      with pytest.raises(RuntimeError, match='same leaf'):
        call(x, w, b)
      with torch.no_grad():
        z = call(x, w, b)                                                # (nothing to hand over)
    g.replay()
    assert torch.equal(z, y), name
    del y
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      got = torch.autograd.grad(call(x, w, b), leaves, dy)
    for _ in range(2):
      for t in got:
        t.fill_(7.0)
      g.replay()
      torch.cuda.synchronize()
      assert all(torch.equal(p, q) for p, q in zip(got, want)), name


@gpu
def test_gradients_go_into_registered_sinks():
  from sg2im_amd import functional as HF
  from sg2im_amd.optim import FlatParams
  import torch.nn as nn

  class Block(nn.Module):
    def __init__(self):
      super().__init__()
      self.norm, self.fc = nn.GroupNorm(4, 32), nn.Linear(32, 24)

    def forward(self, x):
      h = HF.GroupNormAct.apply(x, self.norm.weight, self.norm.bias, 4, 0.2)
      return HF.LinearResidual.apply(h, self.fc.weight, self.fc.bias, None, 0.2)
  m = Block().cuda()
  x, dy = gen(30)(2, 5, 5, 32), gen(31)(2, 5, 5, 24)
  want = torch.autograd.grad(m(x), list(m.parameters()), dy)
  flat = FlatParams(m)
  try:
    flat.grad.zero_()
    for _ in range(2):
      m(x).backward(dy)
    views = [HF._sink(p) for p in m.parameters()]
    for v, g in zip(views, want):
      assert v is not None
      check(v.view(g.shape), 2 * g.to(F64), 4 * u32 * g.abs().to(F64) + 1e-30, 'sink')
  finally:
    flat.close()


# ---- more than 2^31 values --------------------------------------------------------------------------------------------

@gpu
def test_group_norm_and_pack_past_32_bit_offsets():
  """the same image over and over: every image is computed alike, whatever its offset"""
  from sg2im_amd import ops
  r = gen(40)
  one = r(1, 1024, 1024, 64).to(BF16)
  n = 33                                                   # 33 * 2^26 values = 2.2e9
  x = one.expand(n, -1, -1, -1).contiguous()
  w, b = (1 + 0.1 * r(64)).to(BF16), (0.1 * r(64)).to(BF16)
  y, st, p = ops.group_norm_act_forward(x, w, b, 8, 0.2, 1e-5, pack=True)
  assert torch.equal(y[n - 1], y[0]) and torch.equal(st[n - 1], st[0])
  assert torch.equal(p.codes[n - 1], p.codes[0]) and torch.equal(p.exps[n - 1], p.exps[0])
  assert torch.equal(ops.unpack8(p)[n - 1], eight(one[0])[0].to(BF16))
  q = ops.pack8(x)
  assert torch.equal(q.codes[n - 1], p.codes[0]) and torch.equal(q.exps[n - 1], p.exps[0])
  dy = r(1, 1024, 1024, 64).to(BF16).expand(n, -1, -1, -1).contiguous()
  for src in (x, p):
    dx = ops.group_norm_act_backward(dy, src, w, b, 8, 0.2, st)
    assert torch.equal(dx[n - 1], dx[0]) and bool(dx[n - 1].isfinite().all())
    del dx


@gpu
def test_linear_past_32_bit_offsets():
  """rows repeated with a period: every row is computed alike, whatever its offset"""
  from sg2im_amd import ops
  r = gen(41)
  period = 4096
  rows = r(period, 64).to(BF16)
  times = 8448                                             # 8448 * 4096 * 64 = 2.2e9 values
  x = rows.repeat(times, 1)
  w, b = (r(64, 64) / 8).to(BF16), r(64).to(BF16)
  y, signs = ops.linear_forward(x, w, b, x, 0.2, signs=True)
  z, s0 = ops.linear_forward(rows, w, b, rows, 0.2, signs=True)
  assert torch.equal(y[-period:], z) and torch.equal(signs[-period:], s0)
  for gate in (None, signs):
    dx = ops.linear_backward_data(y, w, gate, 0.2)
    assert torch.equal(dx[-period:], dx[:period])
  # the last rows' part of dW and db, added to those of everything before them
  cut = x.size(0) - period
  dw, db = torch.empty(64, 64, device='cuda'), torch.empty(64, device='cuda')
  ops.linear_backward_weight(y, ops.pack8(x), dw, dbias=db, signs=signs, slope=0.2)
  d2, b2 = torch.empty_like(dw), torch.empty_like(db)
  ops.linear_backward_weight(y[:cut], ops.pack8(x[:cut]), d2, dbias=b2, signs=signs[:cut], slope=0.2)
  ops.linear_backward_weight(y[cut:], ops.pack8(x[cut:]), d2, accumulate=True, dbias=b2, bias_accumulate=True, signs=signs[cut:], slope=0.2)
  one = torch.where(sides(s0, 64), z.to(F64), (z.to(F64) * 0.2).to(BF16).to(F64))
  want = times * (one.t() @ eight(rows)[0])
  mag = times * (one.abs().t() @ eight(rows)[0].abs())
  # (a chunk of 64 rows at a time in float32 along a split of at most rows / 64: r / 64 + 64 additions)
  tol = (x.size(0) / 64 + 64 + 256) * u32 * mag
  check(dw, want, tol, 'dweight')
  check(d2, want, tol, 'dweight in two parts')
  unrounded = torch.where(sides(s0, 64), z.to(F64), z.to(F64) * 0.2)
  check(db, times * unrounded.sum(0), (x.size(0) / 64 + 256) * u32 * times * unrounded.abs().sum(0), 'dbias')


# ---- what is refused ------------------------------------------------------------------------------------------------

def test_entry_points_refuse_without_a_gpu():
  from sg2im_amd import _lib
  lib = _lib.load()
  one = ctypes.c_void_p(16)                        # (never dereferenced: every call below is refused before a launch)
  E = _lib.SG2IM_ERR_ARG
  fwd = lambda **k: lib.sg2im_groupnorm_act_forward(*[k.get(n, d) for n, d in (  # noqa: E731
    ('x', one), ('xd', 0), ('n', 1), ('hw', 4), ('c', 8), ('g', 2), ('ga', None), ('be', None), ('pd', 0), ('s', 0.2), ('eps', 1e-5),
    ('y', one), ('yd', 0), ('st', one), ('co', None), ('ex', None), ('ws', one), ('wb', 0), ('stream', None))])
  for bad in (dict(), dict(x=None), dict(g=3), dict(g=0), dict(hw=0), dict(c=0), dict(n=-1), dict(xd=2), dict(yd=5), dict(pd=-1),
              dict(xd=1, yd=0), dict(co=one), dict(eps=-1.0), dict(eps=float('nan')), dict(ws=None, wb=1 << 20)):
    assert fwd(**bad) == E, bad
  assert fwd(n=0) == _lib.SG2IM_OK
  bwd = lambda **k: lib.sg2im_groupnorm_act_backward(*[k.get(n, d) for n, d in (  # noqa: E731
    ('dy', one), ('yd', 0), ('x', one), ('xd', 0), ('co', None), ('ex', None), ('n', 1), ('hw', 4), ('c', 8), ('g', 2), ('ga', None),
    ('be', None), ('pd', 0), ('s', 0.2), ('st', one), ('dx', one), ('dga', None), ('dbe', None), ('gd', 0), ('acc', 0), ('ws', one),
    ('wb', 0), ('stream', None))])
  for bad in (dict(), dict(dy=None), dict(x=None), dict(st=None), dict(g=5), dict(xd=1), dict(ex=one), dict(gd=3), dict(hw=0)):
    assert bwd(**bad) == E, bad
  lin = lambda **k: lib.sg2im_linear_forward(*[k.get(n, d) for n, d in (  # noqa: E731
    ('x', one), ('xd', 0), ('ldx', 8), ('w', one), ('b', None), ('bd', 0), ('r', None), ('ldr', 0), ('s', 0.2), ('y', one), ('yd', 0),
    ('ldy', 8), ('si', None), ('m', 4), ('k', 8), ('n', 8), ('ws', None), ('wb', 0), ('stream', None))])
  for bad in (dict(x=None), dict(w=None), dict(y=None), dict(ldx=7), dict(ldy=7), dict(r=one, ldr=7), dict(k=0), dict(n=0), dict(m=-1),
              dict(m=1 << 31), dict(yd=1), dict(xd=3), dict(bd=2)):
    assert lin(**bad) == E, bad
  assert lin(m=0) == _lib.SG2IM_OK
  assert lib.sg2im_linear_backward_data(one, 0, 7, None, 1.0, one, one, 8, 4, 8, 8, None, 0, None) == E
  for x, ldx, co, wt, bt in ((one, 7, None, 0, 0), (None, 8, one, 0, 0), (one, 8, None, 1, 0), (one, 8, None, 0, 2), (None, 8, None, 0, 0)):
    assert lib.sg2im_linear_backward_weight(one, 0, 8, None, 1.0, x, ldx, co, None, one, wt, 0, one, bt, 0, 4, 8, 8, None, 0, None) == E
  assert lib.sg2im_linear_backward_act(one, 0, 8, None, 0.2, None, 0, one, 0, 0, 4, 8, None, 0, None) == E
  assert lib.sg2im_linear_backward_act(one, 1, 8, None, 0.2, one, 0, None, 0, 0, 4, 8, None, 0, None) == E
  for args in ((None, 0, 4, 8, 8, one, one), (one, 0, 4, 8, 7, one, one), (one, 2, 4, 8, 8, one, one), (one, 0, -1, 8, 8, one, one),
               (one, 0, 4, 0, 8, one, one), (one, 0, 4, 8, 8, None, one)):
    assert lib.sg2im_pack8(*args, None) == E, args
  assert lib.sg2im_unpack8(one, one, 4, 8, None, 0, 8, None) == E


def test_wrappers_refuse_cpu_tensors():
  from sg2im_amd import functional as HF, ops
  x, w = torch.randn(4, 8), torch.randn(6, 8)
  with pytest.raises(TypeError):
    ops.pack8(x)
  with pytest.raises(TypeError):
    HF.LinearResidual.apply(x, w, None, None)
  with pytest.raises(TypeError):
    HF.GroupNormAct.apply(x, None, None, 2)
  with pytest.raises(TypeError):
    ops.unpack8(x)


@gpu
def test_wrappers_refuse():
  from sg2im_amd import functional as HF, ops
  d = 'cuda'
  x, w = torch.randn(4, 8, device=d), torch.randn(6, 8, device=d)
  cases = [
    lambda: HF.GroupNormAct.apply(x, None, None, 3),
    lambda: HF.GroupNormAct.apply(x, torch.ones(7, device=d), None, 2),
    lambda: HF.GroupNormAct.apply(x, torch.ones(8, device=d), torch.ones(8, device=d, dtype=BF16), 2),
    lambda: HF.GroupNormAct.apply(x, torch.ones(8), None, 2),
    lambda: HF.GroupNormAct.apply(x.half(), None, None, 2),
    lambda: HF.GroupNormAct.apply(x.bfloat16(), None, None, 2, 0.2, 1e-5, False, F32),
    lambda: HF.GroupNormAct.apply(x, None, None, 2, 0.2, -1.0),
    lambda: HF.GroupNormAct.apply(x[0], None, None, 2),
    lambda: HF.GroupNormAct.apply(x, None, None, 2, math.inf),
    lambda: HF.LinearResidual.apply(x, w, None, None, math.nan),
    lambda: HF.LinearResidual.apply(x, w, None, None, 1e300),                      # (infinite in float)
    lambda: HF.GroupNormAct.apply(torch.empty(2, 0, 3, 8, device=d), None, None, 2),
    lambda: HF.LinearResidual.apply(x, w[:, :7], None, None),
    lambda: HF.LinearResidual.apply(x, w.bfloat16(), None, None),
    lambda: HF.LinearResidual.apply(x, w, torch.ones(5, device=d), None),
    lambda: HF.LinearResidual.apply(x, w, None, torch.ones(6, device=d)),          # a residual is not broadcast
    lambda: HF.LinearResidual.apply(x, w, None, torch.ones(4, 6, device=d, dtype=BF16)),
    lambda: HF.LinearResidual.apply(x, w, None, None, 1.0, False, BF16),
    lambda: HF.LinearResidual.apply(x.half(), w.half(), None, None),
    lambda: ops.pack8(x.double()),
    lambda: ops.unpack8(ops.pack8(x), torch.float16),
  ]
  for k, f in enumerate(cases):
    with pytest.raises((TypeError, ValueError)):
      f()
      pytest.fail('case %d was taken' % k)
  # no second derivative
  for y in (HF.GroupNormAct.apply(x.requires_grad_(True), None, None, 2), HF.LinearResidual.apply(x, w, None, None)):
    with pytest.raises(RuntimeError):
      torch.autograd.grad(y.sum(), (x,), create_graph=True)
