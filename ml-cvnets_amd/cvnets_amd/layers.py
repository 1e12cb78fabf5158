"""Host-side mirror of ``cvnets.layers`` for the hot path: same class names, constructor signatures,
attribute / sub-module tree and ``state_dict`` keys as the reference, with ``forward`` routed to the HIP
kernels (``cvnets_amd.ops``).  Reference file:line is cited per class.

Because the attribute trees are identical, a model built by the *reference* (``cvnets.get_model``) can be
switched to this implementation by class-swapping its modules in place (see ``cvnets_amd.dropin``).
"""
from __future__ import annotations

import argparse
from typing import Optional, Tuple, Union

import torch
from torch import Tensor, nn

from . import ops, packed

# ---------------------------------------------------------------------------------------------
# opts helpers: the reference reads dotted names off an argparse.Namespace with getattr
# ---------------------------------------------------------------------------------------------


def opt(opts, name: str, default=None):
    return getattr(opts, name, default) if opts is not None else default


def default_opts(**overrides) -> argparse.Namespace:
    """Namespace pre-filled with the model-side values of config/classification/imagenet/mobilevit.yaml."""
    ns = argparse.Namespace()
    base = {
        "model.classification.name": "mobilevit",
        "model.classification.n_classes": 1000,
        "model.classification.classifier_dropout": 0.1,
        "model.classification.mit.mode": "small",
        "model.classification.mit.ffn_dropout": 0.0,
        "model.classification.mit.attn_dropout": 0.0,
        "model.classification.mit.dropout": 0.1,
        "model.classification.mit.number_heads": 4,
        "model.classification.mit.head_dim": None,
        "model.classification.mit.no_fuse_local_global_features": False,
        "model.classification.mit.conv_kernel_size": 3,
        "model.classification.mit.transformer_norm_layer": "layer_norm",
        "model.normalization.name": "batch_norm",
        "model.normalization.momentum": 0.1,
        "model.activation.name": "swish",
        "model.activation.inplace": False,
        "model.activation.neg_slope": 0.1,
        "model.layer.global_pool": "mean",
        "model.classification.vit.mode": "tiny",
        "model.classification.vit.dropout": 0.0,
        "model.classification.vit.norm_layer": "layer_norm",
        "model.classification.vit.no_cls_token": False,
        "model.classification.vit.stochastic_dropout": 0.0,
        "model.classification.vit.sinusoidal_pos_emb": False,
        "model.classification.vit.use_pytorch_mha": False,
        "model.classification.mitv2.width_multiplier": 1.0,
        "model.classification.mitv2.attn_dropout": 0.0,
        "model.classification.mitv2.ffn_dropout": 0.0,
        "model.classification.mitv2.dropout": 0.0,
        "model.classification.mitv2.attn_norm_layer": "layer_norm_2d",
    }
    base.update(overrides)
    for k, v in base.items():
        setattr(ns, k, v)
    return ns


# ---------------------------------------------------------------------------------------------
# activations  (cvnets/layers/activation/{swish,gelu}.py; registry cvnets/layers/activation/__init__.py:15-102)
# ---------------------------------------------------------------------------------------------
class Swish(nn.SiLU):
    def __init__(self, inplace: Optional[bool] = False, *args, **kwargs) -> None:
        super().__init__(inplace=inplace)


class GELU(nn.GELU):
    def __init__(self, *args, **kwargs) -> None:
        super().__init__()


class Identity(nn.Module):
    def forward(self, x):
        return x


class ReLU(nn.ReLU):
    """cvnets/layers/activation/relu.py (the activation of the segmentation heads: model.activation.name = relu)"""

    def __init__(self, inplace: Optional[bool] = False, *args, **kwargs) -> None:
        super().__init__(inplace=bool(inplace))


ACT_FN_REGISTRY = {"swish": Swish, "gelu": GELU, "relu": ReLU}


def build_activation_layer(opts=None, act_type: Optional[str] = None, inplace: Optional[bool] = None, *args, **kwargs) -> nn.Module:
    if act_type is None:
        act_type = opt(opts, "model.activation.name", "swish")
    act_type = act_type.lower()
    if act_type not in ACT_FN_REGISTRY:
        raise NotImplementedError(f"activation '{act_type}' is not on the HIP hot path (supported: {sorted(ACT_FN_REGISTRY)})")
    return ACT_FN_REGISTRY[act_type](inplace=bool(inplace))


def act_code(m: Optional[nn.Module]) -> int:
    if m is None or isinstance(m, (Identity, nn.Identity)):
        return ops.ACT_NONE
    if isinstance(m, nn.SiLU):
        return ops.ACT_SILU
    if isinstance(m, nn.GELU):
        return ops.ACT_GELU
    if isinstance(m, nn.ReLU):
        return ops.ACT_RELU
    raise NotImplementedError(f"activation {m.__class__.__name__} has no HIP kernel")


# ---------------------------------------------------------------------------------------------
# normalisation  (cvnets/layers/normalization/{batch_norm,layer_norm}.py; registry normalization/__init__.py:16-88)
# ---------------------------------------------------------------------------------------------
class BatchNorm2d(nn.BatchNorm2d):
    def __init__(self, num_features: int, eps: Optional[float] = 1e-5, momentum: Optional[float] = 0.1, affine: Optional[bool] = True,
                 track_running_stats: Optional[bool] = True, *args, **kwargs) -> None:
        super().__init__(num_features=num_features, eps=eps, momentum=momentum, affine=affine, track_running_stats=track_running_stats)

    def forward(self, x: Tensor) -> Tensor:
        x = ops.to_nhwc(x)
        training = self.training or not self.track_running_stats
        if self.training and self.track_running_stats and not ops.bn_counters_bumped():
            self.num_batches_tracked.add_(1)  # plumbing (scalar counter)
        return ops.BatchNormAct.apply(x, self.weight, self.bias, self.running_mean, self.running_var,
                                      (ops.ACT_NONE, training, float(self.momentum), float(self.eps)))


class LayerNorm(nn.LayerNorm):
    """cvnets/layers/normalization/layer_norm.py:14-72.  The channel-last branch (:67-68) is cvh_layernorm_*.  The reference's
    channel-first branch (:53-66) is taken whenever ``x.shape[1] == C and x.ndim > 2`` — which also happens, by accident, for a
    [B', S, C] token tensor with S == C (MobileViT-S at 192x192, MobileViT-XXS at 128x128).  That case is reproduced bug-compatibly
    (cvh_ln_seq_*, ``reference_quirk = True``); set ``reference_quirk = False`` for the documented channel-last LayerNorm.  A
    genuine [B, C, H, W] feature map takes the same branch per pixel over its channels (cvh_layernorm_cf_*)."""

    reference_quirk = True

    def __init__(self, normalized_shape, eps: Optional[float] = 1e-5, elementwise_affine: Optional[bool] = True, *args, **kwargs):
        super().__init__(normalized_shape=normalized_shape, eps=eps, elementwise_affine=elementwise_affine)

    def forward(self, x: Tensor) -> Tensor:
        c = self.normalized_shape[0]
        if x.ndim == 3 and x.shape[1] == c and x.shape[2] == c:
            b, s, _ = x.shape
            y = ops.layer_norm_tokens(x.reshape(b * s, c).contiguous(), self, (b, s, 1, 1, s, 1, s))
            return y.view(b, s, c)
        if x.ndim == 4 and x.shape[1] == c:  # a genuine [B, C, H, W] feature map: the channel-first branch (layer_norm.py:53-66)
            if c % 8:
                raise NotImplementedError("channel-first LayerNorm: the NHWC storage pads C to a multiple of 8 (C % 8 == 0 needed)")
            xm = ops.to_nhwc(x)
            b, _, h, w = xm.shape
            gamma = self.weight if self.weight is not None else torch.ones(c, device=xm.device)    # plumbing (elementwise_affine=False)
            beta = self.bias if self.bias is not None else torch.zeros(c, device=xm.device)
            return ops.fmap_of(ops.layer_norm_channel_first(ops.tokens_of(xm), gamma, beta, self.eps), b, h, w)
        if x.ndim > 2 and x.shape[1] == c and x.shape[-1] != c:
            raise NotImplementedError("channel-first LayerNorm is on the HIP hot path for 4-D feature maps (and S == C token tensors) only")
        if x.shape[-1] != c:
            raise NotImplementedError("LayerNorm is supported for channel-last format only")
        shp = x.shape
        y = ops.layer_norm(x.reshape(-1, c), self.weight, self.bias, self.eps)
        return y.view(shp)


class LayerNormFP32(LayerNorm):
    """cvnets/layers/normalization/layer_norm.py:111-137: LayerNorm evaluated in fp32 whatever the activation dtype.  The HIP
    LayerNorm kernel always accumulates statistics and applies the affine in fp32 and rounds once on store, so the two coincide."""


class LayerNorm2D_NCHW(nn.GroupNorm):
    """cvnets/layers/normalization/layer_norm.py:75-108: nn.GroupNorm(num_groups=1) — statistics over (C, H, W) of each sample."""

    def __init__(self, num_features: int, eps: Optional[float] = 1e-5, elementwise_affine: Optional[bool] = True, *args, **kwargs) -> None:
        super().__init__(num_channels=num_features, eps=eps, affine=elementwise_affine, num_groups=1)
        self.num_channels = num_features

    def forward(self, x: Tensor) -> Tensor:
        if x.dim() != 4 or not self.affine:
            raise NotImplementedError("layer_norm_2d is on the HIP hot path for affine 4-D maps only")
        return ops.group_norm1(ops.to_nhwc(x), self.weight, self.bias, self.eps)

    def __repr__(self):
        return "{}(num_channels={}, eps={}, affine={})".format(self.__class__.__name__, self.num_channels, self.eps, self.affine)


NORM_LAYER_REGISTRY = {"batch_norm": BatchNorm2d, "batch_norm_2d": BatchNorm2d, "layer_norm": LayerNorm, "layer_norm_fp32": LayerNormFP32,
                       "layer_norm_2d": LayerNorm2D_NCHW, "layer_norm_nchw": LayerNorm2D_NCHW}


def get_normalization_layer(opts, num_features: int, norm_type: Optional[str] = None, num_groups: Optional[int] = None, *args, **kwargs):
    """cvnets/layers/normalization/__init__.py:35-88 (build_normalization_layer)."""
    if norm_type is None:
        norm_type = opt(opts, "model.normalization.name", "batch_norm")
    momentum = opt(opts, "model.normalization.momentum", 0.1)
    norm_type = norm_type.lower()
    if norm_type not in NORM_LAYER_REGISTRY:
        raise NotImplementedError(f"normalisation '{norm_type}' is not on the HIP hot path (supported: {sorted(NORM_LAYER_REGISTRY)})")
    return NORM_LAYER_REGISTRY[norm_type](normalized_shape=num_features, num_features=num_features, momentum=momentum)


# ---------------------------------------------------------------------------------------------
# conv  (cvnets/layers/conv_layer.py:18-66 Conv2d, :69-277 ConvLayer2d)
# ---------------------------------------------------------------------------------------------
class Conv2d(nn.Conv2d):
    def __init__(self, in_channels: int, out_channels: int, kernel_size, stride=1, padding=0, dilation=1, groups: int = 1, bias: bool = False,
                 padding_mode: str = "zeros", *args, **kwargs) -> None:
        super().__init__(in_channels=in_channels, out_channels=out_channels, kernel_size=kernel_size, stride=stride, padding=padding,
                         dilation=dilation, groups=groups, bias=bias, padding_mode=padding_mode)

    def forward(self, x: Tensor) -> Tensor:
        return _conv_forward(self, None, None, x, self.training)


def _conv_geometry(conv: nn.Conv2d) -> Tuple[int, int, int]:
    if conv.stride[0] != conv.stride[1] or conv.padding[0] != conv.padding[1] or conv.dilation[0] != conv.dilation[1] \
            or conv.kernel_size[0] != conv.kernel_size[1]:
        raise NotImplementedError("anisotropic conv geometry is not on the HIP hot path")
    if conv.padding_mode != "zeros":
        raise NotImplementedError("only zero padding is on the HIP hot path")
    return conv.stride[0], conv.padding[0], conv.dilation[0]


def _conv_forward(conv: nn.Conv2d, norm: Optional[nn.Module], act: Optional[nn.Module], x: Tensor, training: bool,
                  residual: Optional[Tensor] = None, x2: Optional[Tensor] = None) -> Tensor:
    stride, pad, dil = _conv_geometry(conv)
    a = act_code(act)
    use_bn = norm is not None
    stem = conv.groups == 1 and isinstance(norm, nn.BatchNorm2d) and ops.stem_eligible(x, conv.weight, conv.bias, stride, pad, dil, use_bn,
                                                                                        residual, x2)
    if not stem:
        x = ops.to_nhwc(x)
    g = be = rm = rv = None
    momentum, eps, bn_training = 0.1, 1e-5, training
    if use_bn:
        if not isinstance(norm, nn.BatchNorm2d):
            raise NotImplementedError(f"{norm.__class__.__name__} after a conv is not on the HIP hot path")
        g, be, rm, rv = norm.weight, norm.bias, norm.running_mean, norm.running_var
        momentum, eps = norm.momentum, norm.eps
        bn_training = norm.training or not norm.track_running_stats
        if norm.training and norm.track_running_stats and not ops.bn_counters_bumped():
            norm.num_batches_tracked.add_(1)  # plumbing (scalar counter)
    if stem:  # the raw NCHW image batch into the first conv: planes read once, no NHWC repack (csrc/stem.hip)
        return ops.stem_conv_bn_act(x, conv.weight, g, be, rm, rv, act=a, training=bn_training, momentum=momentum, eps=eps)
    if conv.groups == 1:
        return ops.conv_bn_act(x, conv.weight, conv.bias, g, be, rm, rv, stride=stride, pad=pad, dil=dil, act=a, use_bn=use_bn,
                               training=bn_training, momentum=momentum, eps=eps, residual=residual, x2=x2)
    if conv.groups == conv.in_channels == conv.out_channels and conv.bias is None and residual is None and x2 is None:
        return ops.dwconv_bn_act(x, conv.weight, g, be, rm, rv, stride=stride, pad=pad, dil=dil, act=a, use_bn=use_bn,
                                 training=bn_training, momentum=momentum, eps=eps)
    raise NotImplementedError("grouped convs other than depthwise are not on the HIP hot path")


class ConvLayer2d(nn.Module):
    """conv -> norm? -> act? as ``self.block`` (children ``conv``, ``norm``, ``act``); cvnets/layers/conv_layer.py:117-277."""

    def __init__(self, opts, in_channels: int, out_channels: int, kernel_size: Union[int, Tuple[int, int]], stride=1, dilation=1,
                 padding=None, groups: int = 1, bias: bool = False, padding_mode: str = "zeros", use_norm: bool = True, use_act: bool = True,
                 norm_layer: Optional[nn.Module] = None, act_layer: Optional[nn.Module] = None, *args, **kwargs) -> None:
        super().__init__()
        if norm_layer is None and use_norm:
            norm_type = opt(opts, "model.normalization.name", "batch_norm")
            if norm_type == "batch_norm":
                norm_type = "batch_norm_2d"
            norm_layer = get_normalization_layer(opts=opts, num_features=out_channels, norm_type=norm_type)
        if act_layer is None and use_act:
            act_layer = build_activation_layer(opts)
        if use_norm and bias and any(n == "bias" for n, _ in norm_layer.named_parameters()):
            raise AssertionError("Do not use bias when using normalization layers with bias.")
        if use_norm and isinstance(norm_layer, LayerNorm):
            bias = True
        if isinstance(kernel_size, int):
            kernel_size = (kernel_size, kernel_size)
        if isinstance(stride, int):
            stride = (stride, stride)
        if isinstance(dilation, int):
            dilation = (dilation, dilation)
        if padding is None:
            padding = tuple(int((kernel_size[i] - 1) / 2) * dilation[i] for i in range(2))
        if in_channels % groups or out_channels % groups:
            raise ValueError("channels are not divisible by groups")
        block = nn.Sequential()
        conv = Conv2d(in_channels=in_channels, out_channels=out_channels, kernel_size=kernel_size, stride=stride, padding=padding,
                      dilation=dilation, groups=groups, bias=bias, padding_mode=padding_mode)
        block.add_module(name="conv", module=conv)
        self.norm_name = None
        if use_norm:
            block.add_module(name="norm", module=norm_layer)
            self.norm_name = norm_layer.__class__.__name__
        self.act_name = None
        if use_act:
            block.add_module(name="act", module=act_layer)
            self.act_name = act_layer.__class__.__name__
        self.block = block
        self.in_channels = in_channels
        self.out_channels = out_channels
        self.stride = stride
        self.groups = groups
        self.kernel_size = conv.kernel_size
        self.bias = bias
        self.dilation = dilation

    def forward(self, x: Tensor, residual: Optional[Tensor] = None, x2: Optional[Tensor] = None) -> Tensor:
        blk = self.block
        norm = getattr(blk, "norm", None) if "norm" in blk._modules else None
        act = getattr(blk, "act", None) if "act" in blk._modules else None
        return _conv_forward(blk.conv, norm, act, x, self.training, residual=residual, x2=x2)

    def __repr__(self):
        s = self.block[0].__repr__()[:-1]
        if self.norm_name is not None:
            s += ", normalization={}".format(self.norm_name)
        if self.act_name is not None:
            s += ", activation={}".format(self.act_name)
        return s + ")"


# ---------------------------------------------------------------------------------------------
# linear / dropout / pooling  (cvnets/layers/linear_layer.py:17-103, dropout.py:11-29, global_pool.py:16-83)
# ---------------------------------------------------------------------------------------------
class LinearLayer(nn.Module):
    def __init__(self, in_features: int, out_features: int, bias: Optional[bool] = True, channel_first: Optional[bool] = False, *args, **kwargs):
        super().__init__()
        self.weight = nn.Parameter(torch.Tensor(out_features, in_features))
        self.bias = nn.Parameter(torch.Tensor(out_features)) if bias else None
        self.in_features = in_features
        self.out_features = out_features
        self.channel_first = channel_first
        self.reset_params()

    def reset_params(self) -> None:  # linear_layer.py:68-72
        if self.weight is not None:
            torch.nn.init.xavier_uniform_(self.weight)
        if self.bias is not None:
            torch.nn.init.constant_(self.bias, 0)

    def forward(self, x: Tensor, act: int = ops.ACT_NONE, drop_p: float = 0.0, residual: Optional[Tensor] = None) -> Tensor:
        if self.channel_first:
            raise NotImplementedError("channel_first LinearLayer is not on the HIP hot path")
        shp = x.shape
        x2 = x.reshape(-1, shp[-1])
        if x2.dtype != ops.compute_dtype():
            x2 = x2.to(ops.compute_dtype())  # plumbing: only at a dtype boundary
        res2 = residual.reshape(-1, self.out_features) if residual is not None else None
        y = ops.linear(x2.contiguous(), self.weight, self.bias, act=act, drop_p=drop_p, residual=res2)
        return y.view(*shp[:-1], self.out_features)

    def __repr__(self):
        return "{}(in_features={}, out_features={}, bias={}, channel_first={})".format(
            self.__class__.__name__, self.in_features, self.out_features, self.bias is not None, self.channel_first)


class Dropout(nn.Dropout):
    def __init__(self, p: Optional[float] = 0.5, inplace: Optional[bool] = False, *args, **kwargs) -> None:
        super().__init__(p=p, inplace=inplace)

    def forward(self, x: Tensor) -> Tensor:
        return ops.dropout(x, self.p, self.training)


class Dropout2d(nn.Dropout2d):
    """cvnets/layers/dropout.py:32-50"""

    def __init__(self, p: float = 0.5, inplace: bool = False):
        super().__init__(p=p, inplace=inplace)

    def forward(self, x: Tensor) -> Tensor:
        return ops.dropout2d(x, self.p, self.training)


class AdaptiveAvgPool2d(nn.AdaptiveAvgPool2d):
    """cvnets/layers/pooling.py (AdaptiveAvgPool2d): the ASPP image-pooling branch (1) and the PSPNet pyramid bins (1, 2, 3, 6)"""

    def forward(self, x: Tensor) -> Tensor:
        size = self.output_size if isinstance(self.output_size, int) else (self.output_size[0] if self.output_size[0] == self.output_size[1] else None)
        if size is None:
            raise NotImplementedError("non-square adaptive pooling is not on the HIP path")
        return ops.adaptive_avg_pool(x, size)


class UpSample(nn.Upsample):
    """cvnets/layers/upsample.py (nn.Upsample); bilinear only, both corner conventions"""

    def forward(self, x: Tensor) -> Tensor:
        if self.mode != "bilinear":
            raise NotImplementedError("only bilinear up-sampling is on the HIP path")
        H, W = x.shape[-2:]
        if self.size is not None:
            Ho, Wo = (self.size, self.size) if isinstance(self.size, int) else tuple(self.size)
        else:
            sf = self.scale_factor if isinstance(self.scale_factor, (tuple, list)) else (self.scale_factor, self.scale_factor)
            Ho, Wo = int(H * sf[0]), int(W * sf[1])
        return ops.resize_bilinear(ops.to_nhwc(x), Ho, Wo, bool(self.align_corners))


class StochasticDepth(nn.Module):
    """cvnets/layers/stochastic_depth.py:10-18 (torchvision.ops.StochasticDepth): per-sample Bernoulli(1 - p) / (1 - p) scaling; samples run
    along dim 0.  TransformerEncoder fuses it with its residual add (ops.drop_path on the token matrix); this forward is the standalone
    layer for [B, ...] tensors."""

    def __init__(self, p: float, mode: str = "row") -> None:
        super().__init__()
        if mode != "row":
            raise NotImplementedError('only mode="row" (the one the reference constructs) is on the HIP hot path')
        self.p, self.mode = float(p), mode

    def forward(self, x: Tensor) -> Tensor:
        if not self.training or self.p <= 0.0:
            return x
        B = x.shape[0]
        if x.dim() == 4:  # feature map: NHWC rows, one sample = H*W consecutive rows
            x = ops.to_nhwc(x)
            _, C, H, W = x.shape
            y = ops.drop_path(ops.tokens_of(x), None, self.p, True, (B, H * W, 1, 1, H * W, 1, H * W))
            return ops.fmap_of(y, B, H, W)
        C = x.shape[-1]
        rows_per = x.numel() // (B * C)
        x2 = x.reshape(B * rows_per, C)
        if x2.dtype != ops.compute_dtype():
            x2 = x2.to(ops.compute_dtype())
        return ops.drop_path(x2.contiguous(), None, self.p, True, (B, rows_per, 1, 1, rows_per, 1, rows_per)).view(x.shape)

    def __repr__(self) -> str:
        return "{}(p={}, mode={})".format(self.__class__.__name__, self.p, self.mode)


class GlobalPool(nn.Module):
    pool_types = ["mean", "rms", "abs"]

    def __init__(self, pool_type: Optional[str] = "mean", keep_dim: Optional[bool] = False, *args, **kwargs) -> None:
        super().__init__()
        if pool_type != "mean":
            raise NotImplementedError("only mean pooling is on the HIP hot path")
        self.pool_type = pool_type
        self.keep_dim = keep_dim

    def forward(self, x: Tensor) -> Tensor:
        if x.dim() != 4:
            raise NotImplementedError("Currently 2D global pooling supported")
        y = ops.GlobalAvgPool.apply(ops.to_nhwc(x))
        return y.view(y.shape[0], y.shape[1], 1, 1) if self.keep_dim else y

    def __repr__(self):
        return "{}(type={})".format(self.__class__.__name__, self.pool_type)


# ---------------------------------------------------------------------------------------------
# positional embedding  (cvnets/layers/positional_embedding.py:16-180; learnable variant only)
# ---------------------------------------------------------------------------------------------
class LearnablePositionalEmbedding(nn.Module):
    def __init__(self, opts, num_embeddings: int, embedding_dim: int, padding_idx: Optional[int] = None, sequence_first: Optional[bool] = False,
                 interpolation_mode: Optional[str] = "bilinear", *args, **kwargs):
        super().__init__()
        self.pos_embed = nn.Parameter(torch.empty(1, 1, num_embeddings, embedding_dim))
        self.embedding_dim = embedding_dim
        self.num_embeddings = num_embeddings
        self.padding_idx = padding_idx
        self.sequence_first = sequence_first
        self.interpolation_mode = interpolation_mode
        self.reset_parameters()

    def reset_parameters(self) -> None:
        nn.init.trunc_normal_(self.pos_embed, mean=0, std=self.embedding_dim ** -0.5)
        if self.padding_idx is not None:
            with torch.no_grad():
                self.pos_embed[:, :, self.padding_idx, ...] = 0.0

    def table(self, seq_len: int) -> Tensor:
        """the [seq_len, E] float32 table (bilinearly resized along the sequence axis when seq_len differs, positional_embedding.py:90-95);
        the embedding kernels broadcast it over the batch themselves."""
        if self.interpolation_mode != "bilinear":
            raise NotImplementedError("non-bilinear positional embeddings are not on the HIP hot path")
        if self.padding_idx is not None:  # positional_embedding.py:84-86: the padding position is re-zeroed on every call
            with torch.no_grad():
                self.pos_embed[:, :, self.padding_idx, ...] = 0.0
        pe = self.pos_embed.view(self.num_embeddings, self.embedding_dim)
        if seq_len != self.num_embeddings:
            # [N, E] is an NHWC map with H = N, W = 1, C = E: resizing H only is F.interpolate(size=(seq_len, E)) on [1,1,N,E]
            fm = pe.view(1, self.num_embeddings, 1, self.embedding_dim).permute(0, 3, 1, 2)
            pe = ops.resize_bilinear(fm, seq_len, 1).permute(0, 2, 3, 1).reshape(seq_len, self.embedding_dim)
        return pe

    def forward(self, seq_len: int, *args, **kwargs) -> Tensor:
        """reference contract (positional_embedding.py:81-104): [seq_len, 1, E] when sequence_first else [1, seq_len, E]"""
        pe = self.table(seq_len)
        return pe.reshape(seq_len, 1, self.embedding_dim) if self.sequence_first else pe.reshape(1, seq_len, self.embedding_dim)

    def __repr__(self):
        return "{}(num_embeddings={}, embedding_dim={}, padding_idx={}, sequence_first={})".format(
            self.__class__.__name__, self.num_embeddings, self.embedding_dim, self.padding_idx, self.sequence_first)


class PositionalEmbedding(nn.Module):
    def __init__(self, opts, num_embeddings: int, embedding_dim: int, padding_idx: Optional[int] = None, is_learnable: Optional[bool] = False,
                 sequence_first: Optional[bool] = False, interpolation_mode: Optional[str] = "bilinear", *args, **kwargs):
        super().__init__()
        if not is_learnable:
            raise NotImplementedError("sinusoidal positional embeddings are not on the HIP hot path")
        self.pos_embed = LearnablePositionalEmbedding(opts, num_embeddings=num_embeddings, embedding_dim=embedding_dim, padding_idx=padding_idx,
                                                      sequence_first=sequence_first, interpolation_mode=interpolation_mode)

    def table(self, seq_len: int) -> Tensor:
        return self.pos_embed.table(seq_len)

    def forward(self, seq_len: int, *args, **kwargs) -> Tensor:
        return self.pos_embed(seq_len, *args, **kwargs)

    def __repr__(self):
        return self.pos_embed.__repr__()


# ---------------------------------------------------------------------------------------------
# token embedding  (cvnets/layers/embedding.py:15-60)
# ---------------------------------------------------------------------------------------------
class Embedding(nn.Embedding):
    def __init__(self, opts, num_embeddings: int, embedding_dim: int, padding_idx: Optional[int] = None, *args, **kwargs):
        super().__init__(num_embeddings=num_embeddings, embedding_dim=embedding_dim, padding_idx=padding_idx)

    def reset_parameters(self) -> None:
        nn.init.normal_(self.weight, mean=0, std=self.embedding_dim ** -0.5)
        if self.padding_idx is not None:
            nn.init.constant_(self.weight[self.padding_idx], 0)

    def forward(self, tokens: Tensor, pos: Optional[Tensor] = None) -> Tensor:
        """tokens [B, S] -> [B, S, E] (+ pos [S, E] added in the same kernel)"""
        if tokens.dim() != 2:
            raise NotImplementedError("Embedding expects [batch, sequence] token ids on the HIP hot path")
        y = ops.EmbedLookup.apply(tokens, self.weight, pos, self.padding_idx, ops.compute_dtype())
        return y.view(tokens.shape[0], tokens.shape[1], self.embedding_dim)


# ---------------------------------------------------------------------------------------------
# linear self-attention  (cvnets/layers/linear_attention.py:15-215)
# ---------------------------------------------------------------------------------------------
class LinearSelfAttention(nn.Module):
    """MobileViTv2 separable self-attention.  ``forward(x)`` takes the FEATURE MAP [B, C, H, W] (NHWC strides), not the unfolded
    [B, C, P, N] tensor of the reference: pixels with equal (h % patch_h, w % patch_w) are the reference's dim-2 slice, the
    softmax / context sum run over the patches inside the kernel (csrc/linattn.hip), so unfold / fold never materialise.
    qkv_proj's weight rows are consumed in the order key | value | query | 7 zero rows (a 16-byte aligned GEMM output);
    the permutation is an autograd-visible torch.cat of the [1+2C, C] parameter, so its gradient lands in reference order."""

    def __init__(self, opts, embed_dim: int, attn_dropout: Optional[float] = 0.0, bias: Optional[bool] = True, *args, **kwargs) -> None:
        super().__init__()
        self.qkv_proj = ConvLayer2d(opts=opts, in_channels=embed_dim, out_channels=1 + (2 * embed_dim), bias=bias, kernel_size=1,
                                    use_norm=False, use_act=False)
        self.qkv_proj.block.conv._cvh_skip_pack = True
        self.attn_dropout = Dropout(p=attn_dropout)
        self.out_proj = ConvLayer2d(opts=opts, in_channels=embed_dim, out_channels=embed_dim, bias=bias, kernel_size=1, use_norm=False,
                                    use_act=False)
        self.embed_dim = embed_dim

    def __repr__(self):
        return "{}(embed_dim={}, attn_dropout={})".format(self.__class__.__name__, self.embed_dim, self.attn_dropout.p)

    def forward(self, x: Tensor, x_prev: Optional[Tensor] = None, patch_hw: Tuple[int, int] = (2, 2), residual: Optional[Tensor] = None,
                *args, **kwargs) -> Tensor:
        if self.attn_dropout.p > 0.0 and self.training:
            raise NotImplementedError("dropout on the context scores is not on the HIP hot path (mitv2.attn_dropout defaults to 0)")
        C = self.embed_dim
        conv = self.qkv_proj.block.conv
        w, b = conv.weight, conv.bias
        if x_prev is not None:
            # _forward_cross_attn (linear_attention.py:163-207): query and key are projected from x_prev, the value from x; the softmax and
            # the context sum run over the previous frame's patches.  x_prev arrives as the previous frame's FEATURE MAP (the caller folds
            # the reference's [B, C, P, M] tensor); with M == N the fused kernel takes [key(x_prev) | value(x) | query(x_prev)] as it takes
            # the self-attention projection - two GEMMs and a channel concatenation (torch plumbing) instead of one GEMM.
            xp = ops.to_nhwc(x_prev)
            if tuple(xp.shape) != tuple(x.shape):
                raise NotImplementedError("linear cross-attention on the HIP path needs x_prev with the current frame's patch grid (M == N)")
            wkq = torch.cat((w[1:C + 1], w[:1], w.new_zeros((7,) + tuple(w.shape[1:]))), dim=0)  # plumbing: [C+8, C, 1, 1]: key | query | 0
            bkq = torch.cat((b[1:C + 1], b[:1], b.new_zeros(7)), dim=0) if b is not None else None
            kq = ops.conv_bn_act(xp, wkq, bkq)
            v = ops.conv_bn_act(ops.to_nhwc(x), w[C + 1:], b[C + 1:] if b is not None else None)
            kvq = torch.cat((kq[:, :C], v, kq[:, C:]), dim=1).contiguous(memory_format=torch.channels_last)  # plumbing
        else:
            wp = torch.cat((w[1:], w[:1], w.new_zeros((7,) + tuple(w.shape[1:]))), dim=0)  # plumbing: [2C+8, C, 1, 1] row permutation
            bp = torch.cat((b[1:], b[:1], b.new_zeros(7)), dim=0) if b is not None else None
            kvq = ops.conv_bn_act(ops.to_nhwc(x), wp, bp)
        out = ops.linear_attention(kvq, C, patch_hw[0], patch_hw[1])
        return self.out_proj(out, residual=residual)


# ---------------------------------------------------------------------------------------------
# multi-head attention  (cvnets/layers/multi_head_attention.py:18-309)
# ---------------------------------------------------------------------------------------------
class MultiHeadAttention(nn.Module):
    def __init__(self, embed_dim: int, num_heads: int, attn_dropout: Optional[float] = 0.0, bias: Optional[bool] = True,
                 output_dim: Optional[int] = None, coreml_compatible: Optional[bool] = False, *args, **kwargs) -> None:
        if output_dim is None:
            output_dim = embed_dim
        super().__init__()
        if embed_dim % num_heads != 0:
            raise ValueError(f"Embedding dim must be divisible by number of heads. Got: embed_dim={embed_dim} and num_heads={num_heads}")
        self.qkv_proj = LinearLayer(in_features=embed_dim, out_features=3 * embed_dim, bias=bias)
        self.attn_dropout = Dropout(p=attn_dropout)
        self.out_proj = LinearLayer(in_features=embed_dim, out_features=output_dim, bias=bias)
        self.head_dim = embed_dim // num_heads
        self.scaling = self.head_dim ** -0.5
        self.softmax = nn.Softmax(dim=-1)
        self.num_heads = num_heads
        self.embed_dim = embed_dim
        self.coreml_compatible = coreml_compatible
        self.use_separate_proj_weight = embed_dim != output_dim

    def __repr__(self):
        return "{}(head_dim={}, num_heads={}, attn_dropout={})".format(self.__class__.__name__, self.head_dim, self.num_heads, self.attn_dropout.p)

    def forward_tokens(self, x2d: Tensor, seqmap, causal: bool = False, key_padding_mask: Optional[Tensor] = None, out_drop_p: float = 0.0,
                       residual: Optional[Tensor] = None, attn_bias: Optional[Tensor] = None, seqs: Optional[packed.PackedSeqs] = None) -> Tensor:
        """qkv projection -> fused attention -> output projection (+dropout +residual in its epilogue).  `seqs`: the rows are packed sequences
        of these lengths instead of those of `seqmap`."""
        qkv = ops.linear(x2d, self.qkv_proj.weight, self.qkv_proj.bias)
        if seqs is not None:
            if key_padding_mask is not None or attn_bias is not None or (self.training and self.attn_dropout.p > 0.0):
                raise NotImplementedError("packed sequences take no key padding mask, no attention mask and no dropout on the attention probabilities")
            o = packed.attention_qkv(qkv, self.num_heads, seqs, causal=causal)
            return ops.linear(o, self.out_proj.weight, self.out_proj.bias, drop_p=out_drop_p, residual=residual)
        # attn_dropout (multi_head_attention.py:217-218) acts on the softmax output inside the fused kernel; the mask is regenerated in backward
        o = ops.attention(qkv, self.num_heads, seqmap, causal=causal, key_padding_mask=key_padding_mask,
                          drop_p=float(self.attn_dropout.p) if self.training else 0.0, attn_bias=attn_bias)
        return ops.linear(o, self.out_proj.weight, self.out_proj.bias, drop_p=out_drop_p, residual=residual)

    def forward(self, x_q: Tensor, x_kv: Optional[Tensor] = None, key_padding_mask: Optional[Tensor] = None,
                attn_mask: Optional[Tensor] = None, *args, **kwargs) -> Tensor:
        if self.coreml_compatible:
            # forward_tracing (multi_head_attention.py:81-133) is the same product written head by head for export, WITHOUT the two masks
            # (it never reads them): the fused kernels compute it; the masks are dropped exactly as the reference's branch drops them
            key_padding_mask = attn_mask = None
        if x_kv is not None:
            if kwargs.get("use_pytorch_mha", False):
                # (forward_pytorch takes [S, B, C]; the cross-attention path below is batch-first: refuse instead of misreading the axes)
                raise NotImplementedError("cvnets_amd MultiHeadAttention: use_pytorch_mha together with x_kv (sequence-first cross-attention)")
            return self._forward_cross(x_q, x_kv, key_padding_mask, attn_mask)
        seq_first = bool(kwargs.get("use_pytorch_mha", False))
        if seq_first:
            # forward_pytorch (multi_head_attention.py:241-273): F.multi_head_attention_forward on the SAME weights, input [S, B, C]; the
            # kernels gather batch-first sequences, so the tensor is transposed on the way in and out (plumbing copies: not a path any shipped
            # model takes)
            x_q = x_q.transpose(0, 1)
        b, s, c = x_q.shape
        causal, bias = False, None
        if attn_mask is not None:
            causal, bias = _split_mask(attn_mask, b, s, s, allow_2d=seq_first)
        x2 = x_q.reshape(b * s, c)
        if x2.dtype != ops.compute_dtype():
            x2 = x2.to(ops.compute_dtype())
        y = self.forward_tokens(x2.contiguous(), (b, s, 1, 1, s, 1, s), causal=causal, key_padding_mask=key_padding_mask, attn_bias=bias)
        y = y.view(b, s, -1)
        return y.transpose(0, 1) if seq_first else y


def _cross_attention(self, x_q: Tensor, x_kv: Tensor, key_padding_mask: Optional[Tensor], attn_mask: Optional[Tensor]) -> Tensor:
    """Cross-attention (multi_head_attention.py:158-185: query from x_q [N, S, C] with the first C rows of qkv_proj, key / value from x_kv
    [N, T, C] with the other 2C).  Not a path of any §8 model (the spatio-temporal MobileViT uses it), so it is built from the hot path's
    pieces rather than given kernels of its own: two projection GEMMs, the packed [q | k | v] matrix the fused attention kernels take
    (column layout identical to self-attention), both sequences padded to L = max(S, T) with the padded keys marked dead in the key-padding
    table the kernels already honour; the concatenation / padding copies are torch plumbing and differentiate themselves."""
    b, s_len, c = x_q.shape
    t_len = x_kv.shape[1]
    mask_bias = None
    if attn_mask is not None:  # [N, S, T] additive mask (multi_head_attention.py:197-208), padded to the [L, L] square the kernels index
        _, mask_bias = _split_mask(attn_mask, b, s_len, t_len, detect_causal=False)
        Lm = max(s_len, t_len)
        if mask_bias.shape[-2] != Lm or mask_bias.shape[-1] != Lm:
            mask_bias = torch.nn.functional.pad(mask_bias, (0, Lm - t_len, 0, Lm - s_len))  # plumbing; padded keys are dead, padded queries dropped
    if x_kv.shape[0] != b or x_kv.shape[2] != c:
        raise AssertionError(f"x_kv must be [{b}, T, {c}]. Got: {list(x_kv.shape)}")
    dt, d = ops.compute_dtype(), self.embed_dim
    w, bias = self.qkv_proj.weight, self.qkv_proj.bias
    q = ops.linear(x_q.reshape(b * s_len, c).to(dt).contiguous(), w[:d], None if bias is None else bias[:d])
    kv = ops.linear(x_kv.reshape(b * t_len, c).to(dt).contiguous(), w[d:], None if bias is None else bias[d:])
    L = max(s_len, t_len)
    q3, kv3 = q.view(b, s_len, d), kv.view(b, t_len, 2 * d)
    if s_len < L:
        q3 = torch.nn.functional.pad(q3, (0, 0, 0, L - s_len))
    kpm = key_padding_mask
    if kpm is not None and list(kpm.shape) != [b, t_len]:
        raise AssertionError(f"Key_padding_mask should be 2-dimension with shape [{b}, {t_len}]. Got: {list(kpm.shape)}")
    if t_len < L:
        kv3 = torch.nn.functional.pad(kv3, (0, 0, 0, L - t_len))
        dead = torch.zeros(b, L, dtype=torch.bool, device=x_q.device)
        dead[:, t_len:] = True
        if kpm is not None:
            dead[:, :t_len] = kpm.to(torch.bool)
        kpm = dead
    qkv = torch.cat([q3, kv3], dim=-1).reshape(b * L, 3 * d)  # plumbing
    o = ops.attention(qkv, self.num_heads, (b, L, 1, 1, L, 1, L), causal=False, key_padding_mask=kpm,
                      drop_p=float(self.attn_dropout.p) if self.training else 0.0, attn_bias=mask_bias)
    o = o.view(b, L, d)[:, :s_len].reshape(b * s_len, d)
    return ops.linear(o.contiguous(), self.out_proj.weight, self.out_proj.bias).view(b, s_len, -1)


MultiHeadAttention._forward_cross = _cross_attention


def _split_mask(attn_mask: Tensor, b: int, s: int, t: int, allow_2d: bool = False, detect_causal: bool = True):
    """(causal, bias) for an additive attention mask [N, S, T] (multi_head_attention.py:197-208; `allow_2d`: the [S, S] form
    F.multi_head_attention_forward takes, boolean masks included).  The CLIP text tower's causal mask
    (cvnets/text_encoders/transformer.py:343-352) is recognised and GENERATED in-kernel (no mask traffic); any other mask is handed to the
    kernels as a float32 bias tile source."""
    if allow_2d and list(attn_mask.shape) == [s, t]:
        m = attn_mask
    elif list(attn_mask.shape) == [b, s, t]:
        m = attn_mask
    else:
        raise AssertionError(f"Shape of attention mask should be [{b}, {s}, {t}]. Got: {attn_mask.shape}")
    if m.dtype == torch.bool:
        m = torch.zeros(m.shape, dtype=torch.float32, device=m.device).masked_fill(m, float("-inf"))
    if detect_causal and s == t:
        ref = torch.full((s, s), float("-inf"), device=m.device, dtype=m.dtype).triu(1)
        if torch.equal(m, ref.expand_as(m)):
            return True, None
    return False, m.to(torch.float32)
