"""Networks that use the group norm, the residual linear layers and the 8-bit checkpoints: the refinement network with
normalization='group', build_cnn with group norms and M tokens, a training iteration with both.

Reference: the same network in torch on the CPU, in 64 bits, with backward passes written from the definitions (an 8-bit
checkpoint included).  Criterion, as for the other networks of this suite: the relative distance of every tensor is at most
1e-4, or three times the distance of the same reference run in float32 - a LeakyReLU's side may differ where float32 and
64 bits round apart, and that is the same for both.

With 8-bit checkpoints the bound is 1e-3.  A code of a computed activation h differs where float32's error D moves h over a
rounding border: for a share 2 D / s of the elements, with s the block's step, and each of these is then off by s.  Relative to
the root mean square r of h that is sqrt(2 D / s) s / r = sqrt(2 (D / r) (s / r)).  D / r: three layers of sums of some 300
products, sqrt(300) 2^-24 each and a factor two for their amplification by the norms, 6e-6; s / r: at most 2 max|h| / 127
with max|h| <= 4 r, 0.063.  Together 9e-4."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

gpu = pytest.mark.gpu


def eight(x):
  """values of the 8-bit form of x (..., C) in x's type"""
  C = x.size(-1)
  out = torch.empty_like(x)
  for c in range(0, C, 32):
    b = x[..., c:c + 32]
    m, k = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = torch.where(m <= 127.0 / 128.0, k - 7, k - 6)
    e = torch.where(m == 0, torch.full_like(e, -126), e)
    s = torch.ldexp(torch.ones_like(m), e)
    out[..., c:c + 32] = torch.round(b / s) * s
  return out


class GroupRef(torch.autograd.Function):
  @staticmethod
  def forward(ctx, x, w, b, groups, slope, eps, ck):        # x NHWC
    N, C = x.size(0), x.size(-1)
    v = x.reshape(N, -1, groups, C // groups)
    mean = v.mean((1, 3), keepdim=True)
    rstd = ((v - mean).square().mean((1, 3), keepdim=True) + eps).rsqrt()
    ctx.save_for_backward(eight(x) if ck else x, w, b, mean, rstd)
    ctx.g = (groups, slope)
    z = (v - mean) * rstd * w.view(groups, -1) + b.view(groups, -1)
    return torch.where(z > 0, z, z * slope).view_as(x)

  @staticmethod
  def backward(ctx, dy):
    x, w, b, mean, rstd = ctx.saved_tensors
    groups, slope = ctx.g
    N, C = x.size(0), x.size(-1)
    v, g = x.reshape(N, -1, groups, C // groups), dy.reshape(N, -1, groups, C // groups)
    xh, w2 = (v - mean) * rstd, w.view(groups, -1)
    dz = torch.where(xh * w2 + b.view(groups, -1) > 0, g, g * slope)
    gz = dz * w2
    dx = rstd * (gz - gz.mean((1, 3), keepdim=True) - xh * (gz * xh).mean((1, 3), keepdim=True))
    return dx.view_as(x), (dz * xh).sum((0, 1)).view(-1), dz.sum((0, 1)).view(-1), None, None, None, None


class LinearRef(torch.autograd.Function):
  @staticmethod
  def forward(ctx, x, w, b, slope, ck):
    z = x @ w.t() + b
    ctx.save_for_backward(eight(x) if ck else x, w, z)
    ctx.slope = slope
    return torch.where(z > 0, z, z * slope)

  @staticmethod
  def backward(ctx, dy):
    x, w, z = ctx.saved_tensors
    dz = torch.where(z > 0, dy, dy * ctx.slope)
    n = dz.reshape(-1, dz.size(-1))
    return dz @ w, n.t() @ x.reshape(-1, x.size(-1)), n.sum(0), None, None


def nhwc(x):
  return x.permute(0, 2, 3, 1).contiguous()


def nchw(x):
  return x.permute(0, 3, 1, 2).contiguous()


def group(x, norm, slope, p, name):
  return nchw(GroupRef.apply(nhwc(x), p[name + '.weight'], p[name + '.bias'], norm.num_groups, slope, norm.eps, norm.checkpoint8))


def ref_layers(mods, x, p, prefix):
  """build_cnn's modules in torch, NCHW, parameters from p"""
  from sg2im_amd.layers import PixelMlp, ResidualBlock
  mods = list(mods)
  i = 0
  while i < len(mods):
    m, name = mods[i], '%s%d' % (prefix, i)
    if isinstance(m, nn.GroupNorm):
      x = group(x, m, mods[i + 1].negative_slope, p, name)
      i += 1
    elif isinstance(m, nn.LeakyReLU):
      x = F.leaky_relu(x, m.negative_slope)
    elif isinstance(m, nn.Conv2d):
      x = F.conv2d(x, p[name + '.weight'], p[name + '.bias'], stride=m.stride, padding=m.padding)
    elif isinstance(m, ResidualBlock):
      x = x + ref_layers(m.net, x, p, name + '.net.')
    elif isinstance(m, PixelMlp):
      h = nhwc(group(x, m.norm, m.slope, p, name + '.norm'))
      h = LinearRef.apply(h, p[name + '.fc1.weight'], p[name + '.fc1.bias'], m.slope, m.checkpoint8)
      x = x + nchw(LinearRef.apply(h, p[name + '.fc2.weight'], p[name + '.fc2.bias'], 1.0, m.checkpoint8))
    elif isinstance(m, nn.AvgPool2d):
      x = F.avg_pool2d(x, m.kernel_size)
    else:
      raise AssertionError(m)
    i += 1
  return x


def ref_refinement(net, layout, p):
  L, H = len(net.refinement_modules), layout.size(2)
  feats = layout.new_zeros(layout.size(0), 1, H >> L, layout.size(3) >> L)
  for i, mod in enumerate(net.refinement_modules):
    feats = F.interpolate(feats, scale_factor=2, mode='nearest')
    f = H // feats.size(2)
    x = torch.cat([F.avg_pool2d(layout, f) if f > 1 else layout, feats], 1)
    feats = ref_layers(mod.net, x, p, 'refinement_modules.%d.net.' % i)
  return ref_layers(net.output_conv, feats, p, 'output_conv.')


def run(fn, module, x, dy, dtype):
  p = {k: v.detach().cpu().to(dtype).requires_grad_(True) for k, v in module.state_dict().items()}
  x = x.detach().cpu().to(dtype).requires_grad_(True)
  y = fn(x, p)
  g = torch.autograd.grad(y, [x] + list(p.values()), dy.cpu().to(dtype))
  return dict(zip(['y', 'x'] + list(p), [y.detach()] + list(g)))


def check_network(module, fn, x, call=None, bound=1e-4):
  """module on the GPU (NCHW in and out through `call`) against fn in 64 bits"""
  module = module.cuda()
  x = x.cuda().requires_grad_(True)
  y = (call or module)(x)
  dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(3)).cuda()
  names = [k for k, _ in module.named_parameters()]
  got = dict(zip(['y', 'x'] + names, [y.detach()] + list(torch.autograd.grad(y, [x] + list(module.parameters()), dy))))
  want, single = run(fn, module, x, dy, torch.float64), run(fn, module, x, dy, torch.float32)
  for k in got:
    a, b = got[k].detach().cpu().double(), want[k].double()
    scale = float(b.norm())
    if k.endswith('.bias') and want[k[:-4] + 'weight'].dim() == 4:
      # A convolution's bias in front of a norm with one channel per group has no gradient: its sum over the pixels cancels,
      # and what is left is the codes' (or float32's) rounding, of which a single differing code is a visible part.  A bias
      # is the weight of an input that is 1 everywhere; it is held to what a weight gets whose input is of order 1.
      w = want[k[:-4] + 'weight']
      scale = max(scale, float(w.norm()) / w[0].numel() ** 0.5)
    if scale == 0.0:
      assert float(a.abs().max()) == 0.0, k
      continue
    e, ref = float((a - b).norm()) / scale, float((single[k].double() - b).norm()) / scale
    assert e <= max(bound, 3 * ref), (k, e, ref)


def through_nhwc(cnn):
  from sg2im_amd import functional as HF
  return lambda x: HF.NhwcToNchw.apply(cnn(HF.NchwToNhwc.apply(x)))


@gpu
@pytest.mark.parametrize('checkpoint8', [False, True])
@pytest.mark.parametrize('arch', ['I3,C3-64-2,M96,C3-48-2', 'I6,C3-32,R,M50,P2,C1-24'])
def test_build_cnn_with_group_norms_and_pixel_mlps(arch, checkpoint8):
  from sg2im_amd.layers import build_cnn
  torch.manual_seed(1)
  cnn, _ = build_cnn(arch, normalization='group', activation='leakyrelu-0.2', pooling='avg', checkpoint8=checkpoint8)
  for k, v in cnn.named_parameters():
    if v.dim() == 1:
      v.data += 0.1 * torch.randn_like(v)
  x = torch.randn(3, 3 if arch.startswith('I3') else 6, 20, 12)
  check_network(cnn, lambda t, p: ref_layers(cnn, t, p, ''), x, through_nhwc(cnn), 1e-3 if checkpoint8 else 1e-4)


@gpu
@pytest.mark.parametrize('checkpoint8', [False, True])
def test_refinement_network_with_group_norm(checkpoint8):
  from sg2im_amd.crn import RefinementNetwork
  torch.manual_seed(2)
  net = RefinementNetwork((24, 64, 48, 32), normalization='group', activation='leakyrelu-0.2', checkpoint8=checkpoint8)
  for k, v in net.named_parameters():
    if v.dim() == 1:
      v.data += 0.1 * torch.randn_like(v)
  check_network(net, lambda t, p: ref_refinement(net, t, p), torch.randn(3, 24, 32, 16),
                bound=1e-3 if checkpoint8 else 1e-4)


@gpu
def test_pixel_mlp_in_bf16_mode_keeps_its_input():
  """bfloat16 operands, float32 in and out: within the operands' rounding of the 64-bit block (K products of two rounded
  values each: 2 * 2^-8 relative to the absolute sums, twice in a row)"""
  from sg2im_amd import ops
  from sg2im_amd.layers import PixelMlp
  torch.manual_seed(4)
  m = PixelMlp(64, 96, 'leakyrelu-0.2').cuda()
  x = torch.randn(2, 8, 8, 64, device='cuda', requires_grad=True)
  keep, ops.CONV_COMPUTE = ops.CONV_COMPUTE, 1
  try:
    y = m(x)
    grads = torch.autograd.grad(y.sum(), [x] + list(m.parameters()))
  finally:
    ops.CONV_COMPUTE = keep
  assert y.dtype == torch.float32 and all(g.dtype == torch.float32 and bool(g.isfinite().all()) for g in grads)
  d = torch.float64
  n = GroupRef.apply(x.detach().to(d), m.norm.weight.to(d), m.norm.bias.to(d), m.norm.num_groups, 0.2, m.norm.eps, False)
  h = F.leaky_relu(n @ m.fc1.weight.to(d).t() + m.fc1.bias.to(d), 0.2)
  want = x.to(d) + h @ m.fc2.weight.to(d).t() + m.fc2.bias.to(d)
  ah = n.abs() @ m.fc1.weight.to(d).abs().t() + m.fc1.bias.to(d).abs()
  tol = 2.0 ** -8 * (5 * ah @ m.fc2.weight.to(d).abs().t())      # (n, W1, h, W2 rounded, and n's own error)
  assert bool(((y.to(d) - want).abs() <= tol + 1e-6).all())


@gpu
@pytest.mark.parametrize('compute', ['f32', 'bf16'])
def test_training_iterations_with_group_norms(compute):
  """the trainer's iteration, eager and as a replayed graph with a padded batch: bit-equal losses and parameters"""
  from sg2im_amd.synthetic import make_vocab, synthetic_batch
  from sg2im_amd.trainer import Trainer
  dev = torch.device('cuda', 0)
  vocab = make_vocab(184, 7)
  batch = tuple(t.to(dev) if torch.is_tensor(t) else t for t in synthetic_batch(4, seed=11))
  arch = 'C4-64-2,M128,C4-128-2'
  kw = dict(generator_kwargs={'layout_noise_dim': 0, 'normalization': 'group', 'checkpoint8': True,
                              'refinement_dims': (128, 64, 64)},
            d_obj_kwargs={'arch': arch, 'normalization': 'group', 'checkpoint8': True},
            d_img_kwargs={'arch': arch, 'normalization': 'group'}, seed=7, bucket=(32, 64), compute_dtype=compute)
  b = Trainer(vocab, dev, use_graphs=True, **kw)
  lb = [Trainer.losses_to_host(b.step(batch)) for _ in range(4)]
  assert b.graph_stats['captures'] == 1 and b.graph_stats['replays'] == 4
  a = Trainer(vocab, dev, use_graphs=False, **kw)
  la = [Trainer.losses_to_host(a.step(batch)) for _ in range(4)]
  for i in range(4):
    for k in la[i]:
      assert la[i][k] == lb[i][k] and la[i][k] == la[i][k], (i, k, la[i][k], lb[i][k])
  for u, v in ((a.flat_g, b.flat_g), (a.flat_do, b.flat_do), (a.flat_di, b.flat_di)):
    assert torch.equal(u.flat, v.flat) and bool(u.flat.isfinite().all())


def test_module_order_and_refusals_without_a_gpu():
  from sg2im_amd.crn import RefinementNetwork
  from sg2im_amd.layers import PixelMlp, SeqCnn, build_cnn, get_normalization_2d
  cnn, c = build_cnn('C3-64-2,M96,R,C3-48', normalization='group')
  assert isinstance(cnn, SeqCnn) and c == 48 and isinstance(cnn[1], PixelMlp)
  assert [type(m).__name__ for m in cnn] == ['Conv2d', 'PixelMlp', 'ResidualBlock', 'GroupNorm', 'LeakyReLU', 'Conv2d']
  assert [get_normalization_2d(n, 'group').num_groups for n in (64, 48, 100, 7, 1)] == [32, 16, 4, 1, 1]
  keys = set(RefinementNetwork((8, 64, 32), normalization='group').state_dict())
  assert 'refinement_modules.0.net.1.weight' in keys and 'refinement_modules.1.net.4.bias' in keys
  with pytest.raises(ValueError):
    build_cnn('M0x', normalization='group')
  with pytest.raises(ValueError):
    RefinementNetwork((8, 64), normalization='layer')
  batchy, _ = build_cnn('C3-64,R', normalization='batch')
  with pytest.raises(NotImplementedError):
    batchy(torch.zeros(1, 4, 4, 3), count=(torch.ones(1, dtype=torch.int32), 1))
