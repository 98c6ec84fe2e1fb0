"""What may and may not be called on group norm + activation, linear + activation + residual and the 8-bit checkpoints: calls
that record or transform operators instead of running them, the framework's own bookkeeping of launches, and calls
at the limits of a launch."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def entry_points():
  """every entry point by name: (call, its float arguments)"""
  from sg2im_amd import functional as HF, ops
  t = lambda *s: torch.ones(*s)  # noqa: E731
  stats, signs = torch.ones(2, 4, 2, dtype=torch.float64), torch.zeros(6, 1, dtype=torch.int32)
  return {
    'group norm': (lambda x, w, b: HF.GroupNormAct.apply(x, w, b, 4, 0.2), [t(2, 3, 8), t(8), t(8)]),
    'group norm, 8 bits': (lambda x, w, b: HF.GroupNormAct.apply(x, w, b, 4, 0.2, 1e-5, True), [t(2, 3, 8), t(8), t(8)]),
    'linear': (lambda x, w, b, r: HF.LinearResidual.apply(x, w, b, r, 0.2), [t(6, 8), t(5, 8), t(5), t(6, 5)]),
    'pack8': (lambda x: ops.pack8(x).codes, [t(6, 8)]),
    'group norm forward': (lambda x, w, b: ops.group_norm_act_forward(x, w, b, 4, 0.2, 1e-5)[0], [t(2, 3, 8), t(8), t(8)]),
    'group norm backward': (lambda dy, x, w, b: ops.group_norm_act_backward(dy, x, w, b, 4, 0.2, stats),
                            [t(2, 3, 8), t(2, 3, 8), t(8), t(8)]),
    'linear forward': (lambda x, w, b, r: ops.linear_forward(x, w, b, r, 0.2)[0], [t(6, 8), t(5, 8), t(5), t(6, 5)]),
    'linear backward act': (lambda dy, db: ops.linear_backward_act(dy, signs, 0.2, F32, db), [t(6, 5), t(5)]),
    'linear backward data': (lambda dz, w: ops.linear_backward_data(dz, w, signs, 0.2), [t(6, 5), t(5, 8)]),
    'linear backward weight': (lambda dz, x, dw, db: ops.linear_backward_weight(dz, x, dw, dbias=db),
                               [t(6, 5), t(6, 8), t(5, 8), t(5)]),
  }


# ---- calls that are followed, not only run ------------------------------------------------------------------------------
# (refused before a device is looked at, so on CPU tensors too; those without a forward gradient get the TypeError of a CPU tensor)

NAMES = ['group norm', 'group norm, 8 bits', 'linear', 'pack8', 'group norm forward', 'group norm backward', 'linear forward',
         'linear backward act', 'linear backward data', 'linear backward weight']


@pytest.mark.parametrize('name', NAMES)
def test_a_forward_gradient_is_refused(name):
  call, args = entry_points()[name]
  assert list(entry_points()) == NAMES
  with pytest.raises(TypeError):
    call(*args)
  for k in range(len(args)):
    for needs in (False, True):
      with fwAD.dual_level():
        a = [t.clone() for t in args]
        a[k] = fwAD.make_dual(a[k].requires_grad_(needs and 'ward' not in name and name != 'pack8'), torch.ones_like(a[k]))
        with pytest.raises(NotImplementedError, match='forward'):
          call(*a)
        with torch.no_grad(), pytest.raises(NotImplementedError, match='forward'):
          call(*a)


@pytest.mark.parametrize('name', NAMES)
def test_a_recorded_call_is_refused(name):
  from torch.fx.experimental.proxy_tensor import make_fx
  call, args = entry_points()[name]
  with pytest.raises(NotImplementedError, match='records'):
    torch.jit.trace(call, tuple(args))
  with pytest.raises(NotImplementedError, match='records'):
    make_fx(call)(*args)
  with pytest.raises(TypeError):                          # (and nothing of it stays behind)
    call(*args)


def test_unpack8_is_refused_in_a_recording():
  from torch.fx.experimental.proxy_tensor import make_fx
  from sg2im_amd import ops
  call = lambda c, e: ops.unpack8(ops.Packed8(c, e, F32))  # noqa: E731
  args = (torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.uint8))
  for record in (lambda: torch.jit.trace(call, args), lambda: make_fx(call)(*args)):
    with pytest.raises(NotImplementedError, match='records'):
      record()


@gpu
def test_forward_gradients_and_recordings_are_refused_on_the_gpu():
  from sg2im_amd import functional as HF
  x, w = torch.randn(6, 32, device='cuda'), torch.randn(32, 32, device='cuda')
  calls = (lambda x, w: HF.GroupNormAct.apply(x, None, None, 4, 0.2), lambda x, w: HF.LinearResidual.apply(x, w, None, x, 0.2))
  for call in calls:
    with fwAD.dual_level(), pytest.raises(NotImplementedError):
      call(fwAD.make_dual(x, w[:6].contiguous()), w)
    with pytest.raises(NotImplementedError):
      torch.jit.trace(call, (x, w))
    # forward over reverse: the gradient that comes in carries one
    xr = x.clone().requires_grad_(True)
    y = call(xr, w)
    with fwAD.dual_level(), pytest.raises(NotImplementedError):
      torch.autograd.grad(y, (xr,), fwAD.make_dual(torch.ones_like(y), torch.ones_like(y)))


@gpu
def test_a_pending_negation_is_carried_out():
  """the imaginary part of a conjugate is a view of the numbers before their sign is turned"""
  from sg2im_amd import functional as HF, ops
  z = torch.complex(torch.randn(64, 2, device='cuda'), torch.randn(64, 2, device='cuda')).conj()
  v = z.imag
  real = -(-v).clone()
  neg = torch._neg_view
  assert v.is_neg() and not real.is_neg() and torch.equal(v, real)
  for f in (lambda t: ops.unpack8(ops.pack8(t)), lambda t: HF.GroupNormAct.apply(t, None, None, 1, 0.2)):
    for take in (lambda t: t, lambda t: t[:, :1], lambda t: t[:1]):
      assert torch.equal(f(take(v)), f(take(real)))
    assert torch.equal(f(neg(-real)), f(real))
  w = torch.randn(3, 1, device='cuda')
  res = torch.randn(64, 3, device='cuda')
  dy = torch.randn(64, 3, device='cuda')
  outs = []
  for x, a, r, g in ((real[:, :1], w, res, dy), (v[:, :1], neg(-w), neg(-res), neg(-dy))):
    leaves = [t.detach().requires_grad_(True) for t in (x, a, r)]
    y = HF.LinearResidual.apply(leaves[0], leaves[1], None, leaves[2], 0.2)
    outs.append([y.detach()] + [t.clone() for t in torch.autograd.grad(y, leaves, g)])
  assert all(torch.equal(p, q) for p, q in zip(*outs))
  # (the single passes take tensors as they lie in memory)
  with pytest.raises(ValueError, match='negation'):
    ops.linear_forward(neg(real), w[:, :1].expand(3, 2).contiguous(), None, None, 1.0)
  with pytest.raises(ValueError, match='negation'):
    HF.GroupNormAct.apply(real, neg(torch.ones(2, device='cuda')), None, 1)


# ---- one group, several workgroups ----------------------------------------------------------------------------------------

# (channels, groups): widths at which groups reach over the border of the channels that one workgroup takes, a narrow last run
# of channels among them (1600 and 1824 float: the last workgroups' groups are fewer than half of the others'), and one at
# which none does
CROSSING = [(1600, 32, F32), (1632, 32, F32), (1824, 32, F32), (1856, 32, F32), (640, 32, F32), (900, 20, F32), (1040, 16, BF16),
            (2080, 32, BF16), (1024, 32, F32)]


@gpu
@pytest.mark.parametrize('images', [4, 32])             # (32: few sums per image, joined by the normalising pass itself)
@pytest.mark.parametrize('channels,groups,dtype', CROSSING)
def test_groups_that_cross_workgroups_have_one_statistic(channels, groups, dtype, images):
  """every group holds the same numbers: its statistics, and what is normalised with them, have to be the same bits whichever
  workgroup joined the sums; and the same call gives the same bits"""
  from sg2im_amd import ops
  g = torch.Generator(device='cuda').manual_seed(channels)
  D = channels // groups
  one = (torch.randn(images, 32, 32, D, device='cuda', generator=g) * 3 + 1).to(dtype)
  x = one.repeat(1, 1, 1, groups)
  dy = torch.randn(images, 32, 32, channels, device='cuda', generator=g).to(dtype)
  first = None
  for _ in range(8):
    y, stats, _ = ops.group_norm_act_forward(x, None, None, groups, 0.2, 1e-5)
    dx = ops.group_norm_act_backward(dy, x, None, None, groups, 0.2, stats)
    assert torch.equal(stats, stats[:, :1].expand_as(stats))
    assert torch.equal(y, y[..., :D].repeat(1, 1, 1, groups))
    if first is None:
      first = (y, stats, dx)
    assert all(torch.equal(a, b) for a, b in zip(first, (y, stats, dx)))
  v = one.to(torch.float64)
  mean, rstd = v.mean((1, 2, 3)), (v.var((1, 2, 3), unbiased=False) + 1e-5).rsqrt()
  # (n values summed in 64 bits: n 2^-53 of the absolute sums, the mean's square taken from the square's mean)
  n, eps = 1024 * D, 2.0 ** -53
  scale = v.square().mean((1, 2, 3))
  assert bool(((first[1][:, 0, 0] - mean).abs() <= n * eps * v.abs().mean((1, 2, 3))).all())
  assert bool(((first[1][:, 0, 1] - rstd).abs() <= 4 * n * eps * scale * rstd ** 3).all())


# ---- many small images ----------------------------------------------------------------------------------------------------

def test_row_wise_batches_are_not_refused():
  """(the workspace query answers 0 for a size that the passes refuse)"""
  from sg2im_amd import _lib
  lib = _lib.load()
  for backward in (0, 1):
    for batch, hw, channels, groups, bf16 in ((131072, 1, 128, 32, 0), (131072, 1, 64, 32, 1), (1 << 24, 1, 32, 4, 1), (1 << 20, 4, 256, 256, 0),
                                              (300000, 1, 4096, 1, 1), (0x7fffffff, 1, 8, 8, 0)):
      assert lib.sg2im_groupnorm_workspace(batch, hw, channels, groups, bf16, backward) > 0, (batch, channels, groups)
    for batch, hw, channels, groups, bf16 in ((1, 1 << 30, 8, 1, 0), (1, 1, 1 << 28, 1, 1), (1, 1, 1 << 28, 1 << 28, 0), (-1, 1, 8, 1, 0), (1, 0, 8, 1, 0)):
      assert lib.sg2im_groupnorm_workspace(batch, hw, channels, groups, bf16, backward) == 0, (batch, channels, groups)


@gpu
@pytest.mark.parametrize('batch,channels,groups,dtype', [(131072, 128, 32, F32), (131072, 64, 4, BF16), (140000, 96, 32, BF16),
                                                         ((1 << 24) + 4096, 32, 2, BF16)])      # (the last: two launches)
def test_row_wise_batches(batch, channels, groups, dtype):
  """rows repeated with a period, against the period's values in 64 bits"""
  from sg2im_amd import ops
  from tests.test_groupnorm_linear_ckpt8 import check, eight, gen, gn_reference, half_step, u32
  period = 4096
  r = gen(channels)
  rows, d = (2 * r(period, channels) + r(channels)).to(dtype), r(period, channels).to(dtype)
  w, b = (1 + 0.2 * r(channels)).to(dtype), (0.2 * r(channels)).to(dtype)
  times, rest = batch // period, batch % period
  x, dy = torch.empty(batch, channels, device='cuda', dtype=dtype), torch.empty(batch, channels, device='cuda', dtype=dtype)
  for full, one in ((x, rows), (dy, d)):
    full[:times * period].view(times, period, channels).copy_(one)
    full[times * period:] = one[:rest]
  for pack in (False, True):
    y, stats, packed = ops.group_norm_act_forward(x, w, b, groups, 0.2, 1e-5, pack=pack)
    dw, db = torch.empty(channels, device='cuda'), torch.empty(channels, device='cuda')
    if dtype == BF16:
      dw, db = dw.to(dtype), db.to(dtype)
    dx = ops.group_norm_act_backward(dy, packed if pack else x, w, b, groups, 0.2, stats, True, dw, db)
    f = gn_reference(rows, eight(rows)[0] if pack else rows, w, b, groups, 0.2, 1e-5, d)
    for got, name, t in ((y, 'y', dtype), (dx, 'dx', dtype)):
      tol = f[name + '_tol'] + half_step(t) * f[name].abs()
      for at in range(0, times, max(1, times // 7)):
        check(got[at * period:(at + 1) * period], f[name], tol, name)
      check(got[(times - 1) * period:times * period], f[name], tol, name)
      check(got[times * period:], f[name][:rest], tol[:rest] if tol.dim() else tol, name)
      # every period is the same bits
      whole = got[:times * period].view(times, -1)
      assert torch.equal(whole, whole[:1].expand_as(whole)), name
    tail = gn_reference(rows[:rest], eight(rows[:rest])[0] if pack else rows[:rest], w, b, groups, 0.2, 1e-5, d[:rest]) if rest else None
    for got, name in ((dw, 'dw'), (db, 'db')):
      want = times * f[name] + (tail[name] if rest else 0)
      tol = times * f[name + '_tol'] + (tail[name + '_tol'] if rest else 0)
      check(got, want, tol + (half_step(dtype) + u32) * want.abs(), name)


# ---- launches are followed ------------------------------------------------------------------------------------------------

def block():
  """a group norm and a linear layer with everything trained: (call, leaves, gradient that comes in)"""
  from sg2im_amd import functional as HF
  g = torch.Generator(device='cuda').manual_seed(5)
  r = lambda *s: torch.randn(*s, device='cuda', generator=g)  # noqa: E731
  leaves = [t.requires_grad_(True) for t in (r(2, 4, 4, 32), r(32), r(32), r(48, 32), r(48))]

  def call(x, gw, gb, w, b):
    return HF.LinearResidual.apply(HF.GroupNormAct.apply(x, gw, gb, 4, 0.2, 1e-5, True), w, b, None, 0.2)
  return call, leaves, r(2, 4, 4, 48)


@gpu
def test_eager_launches_are_counted_in_both_directions_and_captured_ones_are_not():
  from sg2im_amd import _lib
  call, leaves, dy = block()
  seen = [_lib.eager_epoch()]
  y = call(*leaves)
  seen.append(_lib.eager_epoch())
  torch.autograd.grad(y, leaves, dy)
  seen.append(_lib.eager_epoch())
  # (group norm and product; then at least dx, dW and the norm's pass)
  assert seen[1] - seen[0] == 2 and seen[2] - seen[1] >= 3
  del y
  g = torch.cuda.CUDAGraph()
  with torch.cuda.graph(g):
    torch.autograd.grad(call(*leaves), leaves, dy)
  g.replay()
  torch.cuda.synchronize()
  assert _lib.eager_epoch() == seen[2]


@gpu
def test_launches_are_timed_by_kind():
  from sg2im_amd import ops
  call, leaves, dy = block()
  want = [t.clone() for t in torch.autograd.grad(call(*leaves), leaves, dy)]
  ops.TIMER, ops.TIMER_TAG = ops.KernelTimer(), 'mine'
  try:
    got = torch.autograd.grad(call(*leaves), leaves, dy)
    ops.unpack8(ops.pack8(leaves[0].detach()))
    s, tagged = ops.TIMER.summary(), ops.TIMER.summary('mine')
  finally:
    ops.TIMER = ops.TIMER_TAG = None
  assert all(torch.equal(a, b) for a, b in zip(got, want)) and s == tagged
  rows, k, n, e = 32, 32, 48, 2 * 4 * 4 * 32
  for kind in ('igemm_fwd', 'igemm_dgrad', 'igemm_wgrad'):
    assert s[kind]['launches'] == 1 and s[kind]['flops'] == 2.0 * rows * k * n, kind
  bytes8 = e * 33 / 32
  for kind, amount in (('hbm_group_norm_fwd', 8 * e + bytes8), ('hbm_group_norm_bwd', 8 * e + bytes8), ('hbm_pack8', 4 * e + bytes8),
                       ('hbm_unpack8', 4 * e + bytes8)):
    assert s[kind]['launches'] == 1 and s[kind]['flops'] == amount and s[kind]['ms'] > 0, kind
  # and no longer, once nobody asks
  torch.autograd.grad(call(*leaves), leaves, dy)


@gpu
def test_launches_are_printed_while_they_are_traced(monkeypatch, capfd):
  from sg2im_amd import _lib
  call, leaves, dy = block()
  monkeypatch.setattr(_lib, '_TRACE', True)
  torch.autograd.grad(call(*leaves), leaves, dy)
  names = [l.split()[-1] for l in capfd.readouterr().err.splitlines() if l.startswith('[sg2im]')]
  assert names[:2] == ['sg2im_groupnorm_act_forward', 'sg2im_linear_forward'] and names[-1] == 'sg2im_groupnorm_act_backward'
  assert {'sg2im_linear_backward_data', 'sg2im_linear_backward_weight'} <= set(names)
  monkeypatch.setattr(_lib, '_TRACE', False)
  torch.autograd.grad(call(*leaves), leaves, dy)
  assert '[sg2im]' not in capfd.readouterr().err


# ---- maps larger than the caches; sides of the kink -------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('pack', [False, True])
def test_group_norm_beyond_the_caches(pack, dtype, monkeypatch):
  """x and dy of 400 - 550 MB, from 32 times one image: every image like the first, that one against 64 bits, the parameters'
  gradients against 32 times its sums.  A thread adds up rows / 32 chunks / 32 pixel lanes (16 float) in float32 before they
  are joined in 64 bits: 64 (128) values."""
  from sg2im_amd import ops
  from tests import test_groupnorm_linear_ckpt8 as base
  monkeypatch.setattr(base, 'T', 64 if dtype == BF16 else 128)
  r = base.gen(60)
  n, shape, groups = 32, (1, 256, 256, 64), 8
  one, d = (2 * r(*shape) + r(64)).to(dtype), r(*shape).to(dtype)
  w, b = (1 + 0.2 * r(64)).to(dtype), (0.2 * r(64)).to(dtype)
  x, dy = one.expand(n, -1, -1, -1).contiguous(), d.expand(n, -1, -1, -1).contiguous()
  y, stats, packed = ops.group_norm_act_forward(x, w, b, groups, 0.2, 1e-5, pack=pack)
  dw, db = torch.empty(64, device='cuda', dtype=dtype), torch.empty(64, device='cuda', dtype=dtype)
  dx = ops.group_norm_act_backward(dy, packed if pack else x, w, b, groups, 0.2, stats, True, dw, db)
  assert torch.equal(y, y[:1].expand_as(y)) and torch.equal(dx, dx[:1].expand_as(dx)) and torch.equal(stats, stats[:1].expand_as(stats))
  f = base.gn_reference(one, base.eight(one)[0] if pack else one, w, b, groups, 0.2, 1e-5, d)
  half = base.half_step(dtype)
  base.check(y[:1], f['y'], f['y_tol'] + half * f['y'].abs(), 'y')
  base.check(dx[:1], f['dx'], f['dx_tol'] + half * f['dx'].abs(), 'dx')
  base.check(dw, n * f['dw'], n * f['dw_tol'] + (half + base.u32) * n * f['dw'].abs(), 'dweight')
  base.check(db, n * f['db'], n * f['db_tol'] + (half + base.u32) * n * f['db'].abs(), 'dbias')


@gpu
@pytest.mark.parametrize('pack', [False, True])
@pytest.mark.parametrize('channels', [512, 2048, 100])
def test_which_side_of_the_kink_the_backward_pass_takes(channels, pack):
  """slope 0 and a gradient of 2^p at pixel p: the bits of dbias are the sides.  From x they are the forward pass'; from the
  8-bit form they are those of its values, so an element within half a step of the kink may be on the other one."""
  from sg2im_amd import ops
  from tests.test_groupnorm_linear_ckpt8 import eight, gen
  r = gen(channels)
  x, w, b, groups = r(1, 4, 4, channels), 1 + 0.2 * r(channels), 0.2 * r(channels), 4
  dy = (2.0 ** torch.arange(16, device='cuda')).view(1, 4, 4, 1).expand(1, 4, 4, channels).contiguous()
  y, stats, packed = ops.group_norm_act_forward(x, w, b, groups, 0.0, 1e-5, pack=pack)
  db = torch.empty(channels, device='cuda')
  ops.group_norm_act_backward(dy, packed if pack else x, w, b, groups, 0.0, stats, True, None, db)
  got = (db.long().view(1, -1) >> torch.arange(16, device='cuda').view(16, 1) & 1).bool()
  D = channels // groups
  xd, (seen, exps) = x.double().view(16, channels), eight(x)
  per = xd.view(16, groups, D)
  mean, rstd = per.mean((0, 2)), (per.var((0, 2), unbiased=False) + 1e-5).rsqrt()
  spread = lambda v: v.repeat_interleave(D).view(1, channels)  # noqa: E731
  z = lambda v: (v - spread(mean)) * spread(rstd) * w.double() + b.double()  # noqa: E731
  forward = y.view(16, channels) > 0
  assert torch.equal(forward, z(xd) > 0)
  if not pack:
    assert torch.equal(got, forward)
    return
  assert torch.equal(got, z(seen.view(16, channels)) > 0)
  half_step = torch.pow(2.0, exps.double().view(16, -1) - 128).repeat_interleave(32, 1)[:, :channels]
  near = z(xd).abs() <= half_step * spread(rstd) * w.double().abs() * (1 + 1e-12)
  other = got != forward
  assert not bool((other & ~near).any())
  if channels > 100:
    assert bool(other.any())                        # (it does happen: the two passes are not one function's)


# ---- which gradients are asked for; the widest maps -------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize('shape,groups', [((8, 64, 64, 64), 32), ((3, 40, 40, 105), 5), ((4, 4, 4, 256), 8), ((1, 4, 4, 256), 8)])
@pytest.mark.parametrize('pack', [False, True])
def test_each_gradient_alone_is_what_it_is_among_all(shape, groups, pack):
  from sg2im_amd import functional as HF
  g = torch.Generator(device='cuda').manual_seed(9)
  r = lambda *s: torch.randn(*s, device='cuda', generator=g)  # noqa: E731
  C = shape[-1]
  values, dy = (r(*shape), 1 + 0.1 * r(C), 0.1 * r(C)), r(*shape)

  def grads(wanted):
    leaves = [t.clone().requires_grad_(k in wanted) for k, t in enumerate(values)]
    y = HF.GroupNormAct.apply(*leaves, groups, 0.2, 1e-5, pack)
    return torch.autograd.grad(y, [leaves[k] for k in wanted], dy)
  every = grads((0, 1, 2))
  for wanted in ((0,), (1,), (2,), (1, 2), (0, 2), (0, 1)):
    for k, got in zip(wanted, grads(wanted)):
      assert torch.equal(got, every[k]), (wanted, k)


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('shape,groups', [((2, 1, 1, 1 << 20), 1), ((2, 1, 1, 1 << 20), 1 << 18), ((1, 3, 1, 1000003), 1), ((1, 5, 7, 40000), 40000),
                                          ((1, 1, 1, 1 << 24), 64), ((1, 1 << 22, 1, 3), 1)])
def test_the_widest_and_the_longest_maps(shape, groups, dtype, monkeypatch):
  """(float32 additions in a row per thread: rows / 1024 chunks / the pixel lanes, below 64 here)"""
  from sg2im_amd import functional as HF
  from tests import test_groupnorm_linear_ckpt8 as base
  monkeypatch.setattr(base, 'T', 64)
  r = base.gen(61)
  C = shape[-1]
  x0, w0, b0, dy = (2 * r(*shape) + 1).to(dtype), (1 + 0.2 * r(C)).to(dtype), (0.2 * r(C)).to(dtype), r(*shape).to(dtype)
  half = base.half_step(dtype)
  for pack in (False, True):
    x, w, b = (t.clone().requires_grad_(True) for t in (x0, w0, b0))
    y = HF.GroupNormAct.apply(x, w, b, groups, 0.2, 1e-5, pack)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    seen = x0
    if pack:
      seen = base.eight(x0)[0] if C < 100000 else unpacked(x0)
    f = base.gn_reference(x0, seen, w0, b0, groups, 0.2, 1e-5, dy)
    for name, got in (('y', y), ('dx', dx), ('dw', dw), ('db', db)):
      base.check(got, f[name], f[name + '_tol'] + half * f[name].abs(), name)


def unpacked(x):
  """(the definition in base.eight goes block by block: too many here, and pack8 is held to it elsewhere)"""
  from sg2im_amd import ops
  return ops.unpack8(ops.pack8(x), F32)
