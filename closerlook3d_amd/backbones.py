"""Residual backbone and segmentation decode that call the hot path.

`ResNet` / `Bottleneck` follow `pytorch/models/backbones/resnet.py:22-188`; `SceneSegHeadResNet` and
`MultiPartSegHeadResNet` follow `pytorch/models/heads/segmentation_head.py:15-149`: same constructor arguments, same
sub-module names (so reference checkpoints load), same `end_points` dictionary.  They exist here so
the integration tests and the backbone benchmark can run on the GPU box, where the reference tree is
absent; the reference's own files run unchanged on this engine through `drop_in/`.
"""
import torch
import torch.nn as nn

from .local_aggregation_operators import LocalAggregation, _cfg
from . import pt_utils
from .feed_forward import CounterDropout, FeedForwardBlock
from .pt_utils import MaskedMaxPool, MaskedUpsample


def _conv_bn(cin, cout, momentum, relu):
    layers = [nn.Conv1d(cin, cout, kernel_size=1, bias=False), nn.BatchNorm1d(cout, momentum=momentum)]
    if relu:
        layers.append(nn.ReLU(inplace=True))
    return nn.Sequential(*layers)


# A PointWiseMLP bottleneck runs without the [B,C,N] tensors between its layers (fused.pointwise_bottleneck) for layers
# with at least this many values per channel (B * N): below it the BatchNorm tails are single-launch kernels that keep a
# channel in L2 (csrc/bn_relu.hip, bn2_*_small), and there is no round trip to HBM to save.  (The A/B arms of earlier
# rounds -- nn.Conv1d / BatchNorm1d blocks, the concatenating decoder, the layer-by-layer bottleneck -- are installed
# from OUTSIDE the package by scripts/ab/library_arms.py.)
_FUSE_MIN_VALUES = 16384


def run_conv_bn(seq, x, impl='auto', precision='f32', residual=None, shortcut=None):
    """A `_conv_bn` unit (Conv1d + BatchNorm1d [+ ReLU]) -- optionally the tail of a bottleneck: + residual (through the
    `shortcut` unit when given), then ReLU -- through the engine's kernels (fused.conv_bn_act: MFMA convolutions, fused
    BatchNorm / add / ReLU passes, BatchNorm folded into the convolution in inference), or module by module as the
    reference runs it when impl == 'grouped' or the configuration is outside what the kernels cover."""
    relu = len(seq) == 3 or residual is not None
    if impl != 'grouped' and x.is_cuda:
        from . import fused
        y = fused.conv_bn_act(x, seq[0], seq[1], relu=relu, residual=residual,
                              res_conv=shortcut[0] if shortcut is not None else None,
                              res_bn=shortcut[1] if shortcut is not None else None, precision=precision)
        if y is not None:
            return y
    y = seq(x)
    if residual is not None:
        y = torch.relu(y + (shortcut(residual) if shortcut is not None else residual))
    return y


class MultiInputSequential(nn.Sequential):
    def forward(self, *inputs):
        for module in self._modules.values():
            inputs = module(*inputs)
        return inputs


class Bottleneck(nn.Module):
    def __init__(self, in_channels, out_channels, bottleneck_ratio, radius, nsample, config,
                 downsample=False, sampleDl=None, npoint=None):
        super().__init__()
        self.in_channels, self.out_channels, self.downsample = in_channels, out_channels, downsample
        self.impl = _cfg(config, 'cl3d_impl', 'auto')
        self.precision = _cfg(config, 'cl3d_precision', 'f32')
        mid = out_channels // bottleneck_ratio
        if downsample:
            self.maxpool = MaskedMaxPool(npoint, radius, nsample, sampleDl)
        self.conv1 = _conv_bn(in_channels, mid, config.bn_momentum, relu=True)
        self.local_aggregation = LocalAggregation(mid, mid, radius, nsample, config)
        self.conv2 = _conv_bn(mid, out_channels, config.bn_momentum, relu=False)
        self.relu = nn.ReLU(inplace=True)
        if in_channels != out_channels:
            self.shortcut = _conv_bn(in_channels, out_channels, config.bn_momentum, relu=False)
        # beyond the reference: config.cl3d_feed_forward (hidden channels per channel, 0: none) appends a gated feed-forward
        # block over the points' channels, with config.cl3d_feed_forward_dropout in training
        ratio = _cfg(config, 'cl3d_feed_forward', 0)
        self.feed_forward = None if not ratio else FeedForwardBlock(
            out_channels, max(1, int(round(ratio * out_channels))), precision=self.precision,
            dropout=_cfg(config, 'cl3d_feed_forward_dropout', 0.0))

    def forward(self, xyz, mask, features):
        xyz, mask, features = self._bottleneck(xyz, mask, features)
        return xyz, mask, features if self.feed_forward is None else self.feed_forward(features)

    def _bottleneck(self, xyz, mask, features):
        if self.downsample:
            query_xyz, query_mask, identity = self.maxpool(xyz, mask, features)
        else:
            query_xyz, query_mask, identity = xyz, mask, features
        # the whole bottleneck on the engine -- conv1+BN+ReLU, the operator, then conv2 + BN +
        # shortcut (+ its conv and BN) + add + ReLU as MFMA convolutions and fused BatchNorm passes
        shortcut = self.shortcut if self.in_channels != self.out_channels else None
        la = getattr(self.local_aggregation, 'local_aggregation_operator', None)
        if (self.impl != 'grouped' and features.is_cuda and self.training and getattr(la, 'impl', 'auto') != 'grouped'
                and features.shape[0] * features.shape[2] >= _FUSE_MIN_VALUES):
            # ... and, in training, without the [B,C,N] tensors between the bottleneck's layers: conv1's BatchNorm + ReLU
            # ride in the operator's input staging, the operator's own in conv2's (fused.pointwise_bottleneck for the
            # PointWiseMLP, fused.reduce_bottleneck for PosPool / AdaptiveWeight / PseudoGrid)
            from . import fused
            whole = fused.pointwise_bottleneck if type(la).__name__ == 'PointWiseMLP' else fused.reduce_bottleneck
            out = whole(self.conv1, la, self.conv2, shortcut, query_xyz, xyz, query_mask, mask, features, identity,
                        self.precision)
            if out is not None:
                return query_xyz, query_mask, out
        out = run_conv_bn(self.conv1, features, self.impl, self.precision)
        out = self.local_aggregation(query_xyz, xyz, query_mask, mask, out)
        out = run_conv_bn(self.conv2, out, self.impl, self.precision, residual=identity, shortcut=shortcut)
        return query_xyz, query_mask, out


class ResNet(nn.Module):
    def __init__(self, config, input_features_dim, radius, sampleDl, nsamples, npoints,
                 width=144, depth=2, bottleneck_ratio=2):
        super().__init__()
        self.input_features_dim = input_features_dim
        self.impl = _cfg(config, 'cl3d_impl', 'auto')
        self.precision = _cfg(config, 'cl3d_precision', 'f32')
        self._geometry = (radius, sampleDl, list(nsamples), list(npoints), depth > 1)
        self.conv1 = _conv_bn(input_features_dim, width // 2, config.bn_momentum, relu=True)
        self.la1 = LocalAggregation(width // 2, width // 2, radius, nsamples[0], config)
        self.btnk1 = Bottleneck(width // 2, width, bottleneck_ratio, radius, nsamples[0], config)
        # four strided stages: grid size, radius and width double at each one
        for stage in range(4):
            layer = MultiInputSequential()
            sampleDl *= 2
            layer.add_module("strided_bottleneck",
                             Bottleneck(width, 2 * width, bottleneck_ratio, radius, nsamples[stage], config,
                                        downsample=True, sampleDl=sampleDl, npoint=npoints[stage]))
            radius *= 2
            width *= 2
            for i in range(depth - 1):
                layer.add_module(f"bottlneck{i}",  # (sic) the reference's spelling, kept for checkpoints
                                 Bottleneck(width, width, bottleneck_ratio, radius, nsamples[stage + 1], config))
            setattr(self, f"layer{stage + 1}", layer)

    def forward(self, xyz, mask, features, end_points=None):
        if not end_points:
            end_points = {}
        # coordinates-only products (subsampled clouds, ball queries) go ahead on the index stream
        pt_utils.prefetch_geometry(xyz, mask, *self._geometry)
        device = xyz.device
        features = run_conv_bn(self.conv1, features, self.impl, self.precision)
        features = self.la1(xyz, xyz, mask, mask, features)
        xyz, mask, features = self.btnk1(xyz, mask, features)
        end_points['res1_xyz'], end_points['res1_mask'], end_points['res1_features'] = xyz, mask, features
        for stage in range(4):
            xyz, mask, features = getattr(self, f"layer{stage + 1}")(xyz, mask, features)
            end_points[f'res{stage + 2}_xyz'] = xyz
            end_points[f'res{stage + 2}_mask'] = mask
            end_points[f'res{stage + 2}_features'] = features
        pt_utils.join_index_stream(device)
        return end_points


class _UpsampleDecoder(nn.Module):
    """Nearest-neighbour up-sampling decode shared by the two segmentation heads
    (reference heads/segmentation_head.py:32-48,55-73 and :99-115,125-143)."""

    def _engine_options(self, config):
        """`config` (optional, beyond the reference's constructor arguments) carries the engine's two switches to the
        decoder: cl3d_impl ('grouped' = the reference's own dataflow, for validation) and cl3d_precision."""
        self.impl = getattr(config, 'cl3d_impl', 'auto') if config is not None else 'auto'
        self.precision = getattr(config, 'cl3d_precision', 'f32') if config is not None else 'f32'

    def _make_decoder(self, width, base_radius, nsamples):
        for lvl in range(4):
            setattr(self, f"up{lvl}", MaskedUpsample(radius=(8 >> lvl) * base_radius, nsample=nsamples[3 - lvl],
                                                     mode='nearest'))
        bn = 0.1  # the reference's heads use BatchNorm1d's default momentum
        self.up_conv0 = _conv_bn(24 * width, 4 * width, bn, relu=True)
        self.up_conv1 = _conv_bn(8 * width, 2 * width, bn, relu=True)
        self.up_conv2 = _conv_bn(4 * width, width, bn, relu=True)
        self.up_conv3 = _conv_bn(2 * width, width // 2, bn, relu=True)

    def _decode(self, end_points):
        feats = end_points['res5_features']
        for lvl, (fine, coarse) in enumerate(((4, 5), (3, 4), (2, 3), (1, 2))):
            up, seq = getattr(self, f"up{lvl}"), getattr(self, f"up_conv{lvl}")
            geom = (end_points[f'res{fine}_xyz'], end_points[f'res{coarse}_xyz'],
                    end_points[f'res{fine}_mask'], end_points[f'res{coarse}_mask'])
            skip = end_points[f'res{fine}_features']
            out = None
            if feats.is_cuda and self.impl != 'grouped':
                from . import fused  # the level without the concatenated tensor, see fused.decode_level
                out = fused.decode_level(up, *geom, feats, skip, seq[0], seq[1], self.precision)
            if out is None:
                out = run_conv_bn(seq, torch.cat([up(*geom, feats), skip], 1), self.impl, self.precision)
            feats = out
        return feats


def _seg_classifier(width, nout):
    return nn.Sequential(nn.Conv1d(width // 2, width // 2, kernel_size=1, bias=False),
                         nn.BatchNorm1d(width // 2), nn.ReLU(inplace=True),
                         nn.Conv1d(width // 2, nout, kernel_size=1, bias=True))


def _classify(head, feats, impl, precision):
    """A `_seg_classifier`: its Conv1d + BatchNorm1d + ReLU unit through the engine's kernels like every other such unit
    (run_conv_bn) -- besides the fused BatchNorm passes this keeps the step reproducible: the library convolution's weight
    gradient was the one result of a whole captured step that changed from replay to replay (profiles/r04) --
    then the class-logit convolution (13 / <= 6 output channels, with a bias).  Round 6: that one runs on the engine's
    contraction too (f32, the bias added behind it): as an nn.Conv1d its weight gradient was the library's, and in the
    processes where the library picks an atomics-based algorithm it changed from replay to replay -- the strict
    replay-determinism test caught it in the mode WITHOUT any fork (`head.head.3.weight`: 50 bit patterns in 60 replays,
    profiles/r06/gpu_check_summary.txt), which is also what the once-in-ten-runs failure of round 5 was."""
    x = run_conv_bn(head[:3], feats, impl, precision)
    conv = head[3]
    if (impl != 'grouped' and x.is_cuda and x.dtype == torch.float32 and x.dim() == 3 and conv.kernel_size == (1,)
            and conv.stride == (1,) and conv.groups == 1 and conv.weight.dtype == torch.float32):
        from . import fused
        y = fused._Conv1x1.apply(x, conv.weight.view(conv.weight.shape[0], -1), fused.PRECISIONS['f32'])
        return y if conv.bias is None else y + conv.bias[None, :, None]
    return conv(x)


class SceneSegHeadResNet(_UpsampleDecoder):
    """logits (B, num_classes, N).  Reference: heads/segmentation_head.py:15-77."""

    def __init__(self, num_classes, width, base_radius, nsamples, config=None):
        super().__init__()
        self._engine_options(config)
        self.num_classes, self.base_radius, self.nsamples = num_classes, base_radius, nsamples
        self._make_decoder(width, base_radius, nsamples)
        self.head = _seg_classifier(width, num_classes)

    def forward(self, end_points):
        return _classify(self.head, self._decode(end_points), self.impl, self.precision)


class MultiPartSegHeadResNet(_UpsampleDecoder):
    """One part-logit tensor per shape category: [(B, num_parts[i], N)].  Reference: :80-149."""

    def __init__(self, num_classes, width, base_radius, nsamples, num_parts, config=None):
        super().__init__()
        self._engine_options(config)
        self.num_classes, self.base_radius, self.nsamples, self.num_parts = num_classes, base_radius, nsamples, num_parts
        self._make_decoder(width, base_radius, nsamples)
        self.multi_shape_heads = nn.ModuleList(_seg_classifier(width, num_parts[i]) for i in range(num_classes))

    def forward(self, end_points):
        feats = self._decode(end_points)
        return [_classify(head, feats, self.impl, self.precision) for head in self.multi_shape_heads]


class MaskedGlobalAvgPool1d(nn.Module):
    """Mean over the valid points of every cloud.  Reference: heads/classifier.py:6-14."""

    def forward(self, mask, features):
        return features.sum(-1) / mask.sum(-1)[:, None]


class ClassifierResNet(nn.Module):
    """logits (B, num_classes) from `res5_features`.  Reference: heads/classifier.py:17-54 (same layer indices
    inside `classifier`, so checkpoints load unchanged).  `config` (optional, beyond the reference's constructor arguments):
    cl3d_counter_dropout replaces nn.Dropout by the dropout that stores no mask."""

    def __init__(self, num_classes, width, config=None):
        super().__init__()
        dropout = CounterDropout if config is not None and _cfg(config, 'cl3d_counter_dropout', False) else nn.Dropout
        self.num_classes = num_classes
        self.pool = MaskedGlobalAvgPool1d()
        layers, cin = [], 16 * width
        for cout in (8 * width, 4 * width, 2 * width):
            layers += [nn.Linear(cin, cout), nn.BatchNorm1d(cout), nn.ReLU(inplace=True), dropout(0.5)]
            cin = cout
        layers.append(nn.Linear(cin, num_classes))
        self.classifier = nn.Sequential(*layers)

    def forward(self, end_points):
        return self.classifier(self.pool(end_points['res5_mask'], end_points['res5_features']))
