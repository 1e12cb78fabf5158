"""Host-side mirror of ``cvnets.modules`` for the hot path (InvertedResidual, TransformerEncoder, MobileViTBlock):
same constructor signatures, attribute trees and state_dict keys as the reference; forward = HIP kernels.
"""
from __future__ import annotations

import math
import os
from typing import Optional, Tuple, Union

import torch
from torch import Tensor, nn

from . import fused, ops
from .layers import (ConvLayer2d, Dropout, Identity, LayerNorm, LinearLayer, LinearSelfAttention, MultiHeadAttention, StochasticDepth, act_code,
                     build_activation_layer, get_normalization_layer, opt)


_FUSED_FFN_BWD = os.environ.get("CVH_FUSED_FFN_BWD", "1") != "0"  # developer A/B switch
_FUSED_IR = os.environ.get("CVH_FUSED_IR", "1") != "0"  # developer A/B switch: InvertedResidual through BatchNorm links (fused.py)


def set_fused_inverted_residual(flag: bool) -> None:
    global _FUSED_IR
    _FUSED_IR = bool(flag)


def make_divisible(v: Union[float, int], divisor: Optional[int] = 8, min_value: Optional[Union[float, int]] = None) -> Union[float, int]:
    """cvnets/utils/math_utils.py make_divisible (used at cvnets/modules/mobilenetv2.py:176)."""
    if min_value is None:
        min_value = divisor
    new_v = max(min_value, int(v + divisor / 2) // divisor * divisor)
    if new_v < 0.9 * v:
        new_v += divisor
    return new_v


class InvertedResidual(nn.Module):
    """cvnets/modules/mobilenetv2.py:141-246: exp 1x1-BN-act -> depthwise 3x3-BN-act -> red 1x1-BN (+x)."""

    def __init__(self, opts, in_channels: int, out_channels: int, stride: int, expand_ratio: Union[int, float], dilation: int = 1,
                 skip_connection: Optional[bool] = True, *args, **kwargs) -> None:
        assert stride in [1, 2]
        hidden_dim = make_divisible(int(round(in_channels * expand_ratio)), 8)
        super().__init__()
        block = nn.Sequential()
        if expand_ratio != 1:
            block.add_module(name="exp_1x1", module=ConvLayer2d(opts, in_channels=in_channels, out_channels=hidden_dim, kernel_size=1,
                                                                use_act=True, use_norm=True))
        block.add_module(name="conv_3x3", module=ConvLayer2d(opts, in_channels=hidden_dim, out_channels=hidden_dim, stride=stride,
                                                             kernel_size=3, groups=hidden_dim, use_act=True, use_norm=True, dilation=dilation))
        block.add_module(name="red_1x1", module=ConvLayer2d(opts, in_channels=hidden_dim, out_channels=out_channels, kernel_size=1,
                                                            use_act=False, use_norm=True))
        self.block = block
        self.in_channels = in_channels
        self.out_channels = out_channels
        self.exp = expand_ratio
        self.dilation = dilation
        self.stride = stride
        self.use_res_connect = self.stride == 1 and in_channels == out_channels and skip_connection

    def forward(self, x: Tensor, *args, **kwargs) -> Tensor:
        x = ops.to_nhwc(x)
        y = x
        mods = self.block._modules
        if _FUSED_IR and self._fusable():
            # BatchNorm links (cvnets_amd/fused.py): the whole block is one autograd node, no standalone BatchNorm pass on the 4x-wide tensors
            trip = []
            for name in ("exp_1x1", "conv_3x3", "red_1x1"):
                blk = mods[name].block
                norm = blk.norm
                if norm.training and norm.track_running_stats and not ops.bn_counters_bumped():
                    norm.num_batches_tracked.add_(1)  # plumbing (scalar counter)
                trip.append((blk.conv, norm, act_code(getattr(blk, "act", None))))
            return fused.inverted_residual(x, trip[0], trip[1], trip[2], stride=self.stride, use_res=self.use_res_connect)
        if "exp_1x1" in mods:
            y = mods["exp_1x1"](y)
        y = mods["conv_3x3"](y)
        # the residual add rides in the BN-apply pass of the projection conv
        return mods["red_1x1"](y, residual=x if self.use_res_connect else None)

    def _fusable(self) -> bool:
        mods = self.block._modules
        if "exp_1x1" not in mods or self.dilation != 1:
            return False
        modes = set()
        for name in ("exp_1x1", "conv_3x3", "red_1x1"):
            blk = mods[name].block
            conv, norm = getattr(blk, "conv", None), getattr(blk, "norm", None)
            if not isinstance(conv, nn.Conv2d) or conv.bias is not None or not isinstance(norm, nn.BatchNorm2d) or not norm.affine \
                    or norm.momentum is None or (not norm.track_running_stats and not norm.training):
                return False
            if norm.running_mean is None and not norm.training:
                return False
            if conv.weight.shape[1] % 8 and conv.groups == 1:
                return False
            if conv.weight.shape[0] % 8:  # hidden / output widths: the fused kernels move 8-channel (16 B) groups
                return False
            modes.add((bool(norm.training), bool(norm.track_running_stats)))
        dwc = mods["conv_3x3"].block.conv
        if tuple(dwc.kernel_size) != (3, 3) or tuple(dwc.padding) != (1, 1) or dwc.groups != dwc.weight.shape[0]:
            return False  # InvertedResidualFn hard-codes the depthwise 3x3 / pad 1 geometry
        if len(modes) != 1:
            return False  # partially frozen BatchNorm: the fused node takes ONE train / eval mode for all three norms
        return mods["red_1x1"].block._modules.get("act") is None

    def __repr__(self) -> str:
        return "{}(in_channels={}, out_channels={}, stride={}, exp={}, dilation={}, skip_conn={})".format(
            self.__class__.__name__, self.in_channels, self.out_channels, self.stride, self.exp, self.dilation, self.use_res_connect)


class TransformerEncoder(nn.Module):
    """cvnets/modules/transformer.py:26-156 pre-norm block.  ``forward_tokens`` runs it on a [rows, C] token matrix whose
    sequences are described by a seqmap (see ops.AttentionFn); ``forward`` is the reference's [B, S, C] signature."""

    def __init__(self, opts, embed_dim: int, ffn_latent_dim: int, num_heads: Optional[int] = 8, attn_dropout: Optional[float] = 0.0,
                 dropout: Optional[float] = 0.0, ffn_dropout: Optional[float] = 0.0, transformer_norm_layer: Optional[str] = "layer_norm",
                 stochastic_dropout: Optional[float] = 0.0, *args, **kwargs) -> None:
        super().__init__()
        if num_heads <= 1:
            raise NotImplementedError("SingleHeadAttention is not on the HIP hot path")
        attn_unit = MultiHeadAttention(embed_dim, num_heads, attn_dropout=attn_dropout, bias=True,
                                       coreml_compatible=opt(opts, "common.enable_coreml_compatible_module", False))
        self.pre_norm_mha = nn.Sequential(
            get_normalization_layer(opts=opts, norm_type=transformer_norm_layer, num_features=embed_dim),
            attn_unit,
            Dropout(p=dropout),
        )
        act_name = build_activation_layer(opts)
        self.pre_norm_ffn = nn.Sequential(
            get_normalization_layer(opts=opts, norm_type=transformer_norm_layer, num_features=embed_dim),
            LinearLayer(in_features=embed_dim, out_features=ffn_latent_dim, bias=True),
            act_name,
            Dropout(p=ffn_dropout),
            LinearLayer(in_features=ffn_latent_dim, out_features=embed_dim, bias=True),
            Dropout(p=dropout),
        )
        self.drop_path = Identity()
        if stochastic_dropout > 0.0:
            if dropout > 0.0:  # transformer.py:108-112: the reference refuses this combination as well
                raise ValueError("Stochastic dropout and dropout are mutually exclusive. Use either of them, but not both."
                                 " Got: {} and {}".format(stochastic_dropout, dropout))
            self.drop_path = StochasticDepth(p=stochastic_dropout, mode="row")
        self.embed_dim = embed_dim
        self.ffn_dim = ffn_latent_dim
        self.ffn_dropout = ffn_dropout
        self.stochastic_dropout = stochastic_dropout
        self.std_dropout = dropout
        self.attn_fn_name = attn_unit.__class__.__name__
        self.act_fn_name = act_name.__class__.__name__
        self.norm_type = transformer_norm_layer

    def __repr__(self) -> str:
        return "{}(embed_dim={}, ffn_dim={}, dropout={}, ffn_dropout={}, stochastic_dropout={}, attn_fn={}, act_fn={}, norm_fn={})".format(
            self.__class__.__name__, self.embed_dim, self.ffn_dim, self.std_dropout, self.ffn_dropout, self.stochastic_dropout,
            self.attn_fn_name, self.act_fn_name, self.norm_type)

    def forward_tokens(self, x: Tensor, seqmap, causal: bool = False, key_padding_mask: Optional[Tensor] = None,
                       attn_bias: Optional[Tensor] = None, seqs=None) -> Tensor:
        """`seqs` (packed.PackedSeqs): the rows of x are packed sequences; `seqmap` then names no sequences (ops.NO_SEQMAP)"""
        ln1, mha, drop1 = self.pre_norm_mha[0], self.pre_norm_mha[1], self.pre_norm_mha[2]
        if not isinstance(ln1, nn.LayerNorm):
            raise NotImplementedError("transformer_norm_layer must be layer_norm on the HIP hot path")
        p1 = drop1.p if self.training else 0.0
        sd = self.drop_path.p if (self.training and isinstance(self.drop_path, StochasticDepth)) else 0.0
        if sd > 0.0:
            if seqs is not None:
                raise NotImplementedError("stochastic depth on packed sequences")
            # x = x + StochasticDepth(Dropout(branch(LN(x)))): one Bernoulli draw per sample scales the whole branch; the residual add rides in
            # the drop-path kernel instead of the GEMM epilogue (transformer.py:140-155)
            y = ops.layer_norm_tokens(x, ln1, seqmap)
            x = ops.drop_path(mha.forward_tokens(y, seqmap, causal=causal, key_padding_mask=key_padding_mask, out_drop_p=p1, attn_bias=attn_bias), x, sd,
                              True, seqmap)
            return self._ffn_tokens(x, seqmap, sd)
        # x = x + Dropout(MHA(LN(x)))   — dropout and residual live in the out_proj GEMM epilogue; the fork x -> (x, LN(x)) is one autograd
        # node, so the two gradients of x meet inside the LayerNorm backward kernel
        x, y = ops.layer_norm_fork(x, ln1, seqmap)
        x = mha.forward_tokens(y, seqmap, causal=causal, key_padding_mask=key_padding_mask, out_drop_p=p1, residual=x, attn_bias=attn_bias, seqs=seqs)
        return self._ffn_tokens(x, seqmap, 0.0)

    def _ffn_tokens(self, x: Tensor, seqmap, sd: float) -> Tensor:
        """x + StochasticDepth(Dropout(W2 Dropout(act(W1 LN(x)))))   (transformer.py:153-154)"""
        ln2, fc1, act, drop_ffn, fc2, drop2 = (self.pre_norm_ffn[i] for i in range(6))
        p2 = drop2.p if self.training else 0.0
        pf = drop_ffn.p if self.training else 0.0  # ffn_dropout (transformer.py:92; 0.0 in every shipped YAML): un-fused — a standalone pass over the hidden tensor
        if sd > 0.0:
            y = ops.layer_norm_tokens(x, ln2, seqmap)
            h = ops.dropout(ops.linear(y, fc1.weight, fc1.bias, act=act_code(act)), pf, pf > 0.0)
            h = ops.linear(h, fc2.weight, fc2.bias, drop_p=p2)
            return ops.drop_path(h, x, sd, True, seqmap)
        x, y = ops.layer_norm_fork(x, ln2, seqmap)
        a = act_code(act)
        if pf > 0.0:
            h = ops.dropout(ops.linear(y, fc1.weight, fc1.bias, act=a), pf, True)
            return ops.linear(h, fc2.weight, fc2.bias, drop_p=p2, residual=x)
        if _FUSED_FFN_BWD and fc1.out_features >= 1024 and ops.ffn_stores_derivative(y, fc1.weight, a):
            # transformer-sized FFNs (ViT-B: 3072 hidden): fc1's epilogue evaluates erf / exp once and stores GELU'(pre) instead of the
            # pre-activation; fc2's dX GEMM multiplies by it - the separate activation-backward pass over the hidden gradient is gone.
            # (With act'(pre) EVALUATED in the dX epilogue the large-tile GEMM lost 4.5 %: erf / exp serialise behind its MFMA work.)
            h, dv = ops.linear(y, fc1.weight, fc1.bias, act=ops.ACT_GELU_D, expose_pre=True)
            return ops.linear(h, fc2.weight, fc2.bias, drop_p=p2, residual=x, in_pre=dv, in_act=ops.ACT_DERIV)
        if not _FUSED_FFN_BWD or fc1.out_features >= 1024:
            return ops.linear(ops.linear(y, fc1.weight, fc1.bias, act=a), fc2.weight, fc2.bias, drop_p=p2, residual=x)
        h, pre = ops.linear(y, fc1.weight, fc1.bias, act=a, expose_pre=True)
        # fc2's dX GEMM applies act'(pre) in its epilogue and returns the gradient of fc1's pre-activation directly
        return ops.linear(h, fc2.weight, fc2.bias, drop_p=p2, residual=x, in_pre=pre, in_act=a)

    def _forward_cross(self, x: Tensor, x_prev: Tensor, key_padding_mask: Optional[Tensor], attn_mask: Optional[Tensor]) -> Tensor:
        """transformer.py:131-155 with x_kv = x_prev: the query is LN(x), key and value come from x_prev AS GIVEN (the reference does not
        normalise it).  Used by the spatio-temporal MobileViT block only, so it is composed from the hot path's ops (layers.py
        `_cross_attention`) instead of riding the fused epilogues of the self-attention path."""
        ln1, mha, drop1 = self.pre_norm_mha[0], self.pre_norm_mha[1], self.pre_norm_mha[2]
        if not isinstance(ln1, nn.LayerNorm):
            raise NotImplementedError("transformer_norm_layer must be layer_norm on the HIP hot path")
        b, s, c = x.shape
        seqmap = (b, s, 1, 1, s, 1, s)
        x2 = x.reshape(b * s, c)
        if x2.dtype != ops.compute_dtype():
            x2 = x2.to(ops.compute_dtype())
        x2 = x2.contiguous()
        p1 = drop1.p if self.training else 0.0
        sd = self.drop_path.p if (self.training and isinstance(self.drop_path, StochasticDepth)) else 0.0
        y = ops.layer_norm_tokens(x2, ln1, seqmap)
        a = mha(y.view(b, s, c), x_kv=x_prev, key_padding_mask=key_padding_mask, attn_mask=attn_mask).reshape(b * s, c)
        a = ops.dropout(a, p1, p1 > 0.0)
        x2 = ops.drop_path(a, x2, sd, sd > 0.0, seqmap)
        return self._ffn_tokens(x2, seqmap, sd).view(b, s, c)

    def forward(self, x: Tensor, x_prev: Optional[Tensor] = None, key_padding_mask: Optional[Tensor] = None,
                attn_mask: Optional[Tensor] = None, *args, **kwargs) -> Tensor:
        if x_prev is not None:
            return self._forward_cross(x, x_prev, key_padding_mask, attn_mask)
        b, s, c = x.shape
        causal, bias = False, None
        if attn_mask is not None:
            from .layers import _split_mask
            causal, bias = _split_mask(attn_mask, b, s, s)  # the causal triangle is generated in-kernel, any other mask becomes a bias source
        x2 = x.reshape(b * s, c)
        if x2.dtype != ops.compute_dtype():
            x2 = x2.to(ops.compute_dtype())
        y = self.forward_tokens(x2.contiguous(), (b, s, 1, 1, s, 1, s), causal=causal, key_padding_mask=key_padding_mask, attn_bias=bias)
        return y.view(b, s, c)


class MobileViTBlock(nn.Module):
    """cvnets/modules/mobilevit_block.py:19-326.  local_rep (3x3 conv-BN-act, 1x1 conv) -> [unfold] -> L x TransformerEncoder
    -> LayerNorm -> [fold] -> 1x1 conv-BN-act -> 3x3 fusion conv over cat(res, fm).  In NHWC the unfold/fold permutation is
    pure addressing inside the attention kernel and the cat is two source pointers of the fusion conv — neither touches HBM."""

    def __init__(self, opts, in_channels: int, transformer_dim: int, ffn_dim: int, n_transformer_blocks: Optional[int] = 2,
                 head_dim: Optional[int] = 32, attn_dropout: Optional[float] = 0.0, dropout: Optional[int] = 0.0,
                 ffn_dropout: Optional[int] = 0.0, patch_h: Optional[int] = 8, patch_w: Optional[int] = 8,
                 transformer_norm_layer: Optional[str] = "layer_norm", conv_ksize: Optional[int] = 3, dilation: Optional[int] = 1,
                 no_fusion: Optional[bool] = False, *args, **kwargs) -> None:
        conv_3x3_in = ConvLayer2d(opts=opts, in_channels=in_channels, out_channels=in_channels, kernel_size=conv_ksize, stride=1,
                                  use_norm=True, use_act=True, dilation=dilation)
        conv_1x1_in = ConvLayer2d(opts=opts, in_channels=in_channels, out_channels=transformer_dim, kernel_size=1, stride=1,
                                  use_norm=False, use_act=False)
        conv_1x1_out = ConvLayer2d(opts=opts, in_channels=transformer_dim, out_channels=in_channels, kernel_size=1, stride=1,
                                   use_norm=True, use_act=True)
        conv_3x3_out = None
        if not no_fusion:
            conv_3x3_out = ConvLayer2d(opts=opts, in_channels=2 * in_channels, out_channels=in_channels, kernel_size=conv_ksize, stride=1,
                                       use_norm=True, use_act=True)
        super().__init__()
        self.local_rep = nn.Sequential()
        self.local_rep.add_module(name="conv_3x3", module=conv_3x3_in)
        self.local_rep.add_module(name="conv_1x1", module=conv_1x1_in)
        assert transformer_dim % head_dim == 0
        num_heads = transformer_dim // head_dim
        global_rep = [
            TransformerEncoder(opts=opts, embed_dim=transformer_dim, ffn_latent_dim=ffn_dim, num_heads=num_heads, attn_dropout=attn_dropout,
                               dropout=dropout, ffn_dropout=ffn_dropout, transformer_norm_layer=transformer_norm_layer)
            for _ in range(n_transformer_blocks)
        ]
        global_rep.append(get_normalization_layer(opts=opts, norm_type=transformer_norm_layer, num_features=transformer_dim))
        self.global_rep = nn.Sequential(*global_rep)
        self.conv_proj = conv_1x1_out
        self.fusion = conv_3x3_out
        self.patch_h = patch_h
        self.patch_w = patch_w
        self.patch_area = self.patch_w * self.patch_h
        self.cnn_in_dim = in_channels
        self.cnn_out_dim = transformer_dim
        self.n_heads = num_heads
        self.ffn_dim = ffn_dim
        self.dropout = dropout
        self.attn_dropout = attn_dropout
        self.ffn_dropout = ffn_dropout
        self.dilation = dilation
        self.n_blocks = n_transformer_blocks
        self.conv_ksize = conv_ksize

    def forward_spatial(self, x: Tensor) -> Tensor:
        x = ops.to_nhwc(x)
        res = x
        if self.fusion is not None:  # x feeds local_rep AND the fusion concat: their two gradients meet in cvh_add (ops.Fork2)
            x, res = ops.fork2(x)
        fm = self.local_rep.conv_3x3(x)
        fm = self.local_rep.conv_1x1(fm)
        B, d, H, W = fm.shape
        ph, pw = self.patch_h, self.patch_w
        Hn, Wn = int(math.ceil(H / ph) * ph), int(math.ceil(W / pw) * pw)
        interpolate = (Hn != H) or (Wn != W)
        if interpolate:  # reference: bilinear resize to a multiple of the patch (mobilevit_block.py:191-200)
            fm = ops.resize_bilinear(fm, Hn, Wn)
        H0, W0, H, W = H, W, Hn, Wn
        n_h, n_w = H // ph, W // pw
        seqmap = (B * ph * pw, n_h * n_w, ph, pw, n_w, H, W)
        t = ops.tokens_of(fm)
        for layer in self.global_rep:
            if isinstance(layer, TransformerEncoder):
                t = layer.forward_tokens(t, seqmap)
            else:
                if not isinstance(layer, nn.LayerNorm):
                    raise NotImplementedError("transformer_norm_layer must be layer_norm on the HIP hot path")
                t = ops.layer_norm_tokens(t, layer, seqmap)
        fm = ops.fmap_of(t, B, H, W)
        if interpolate:  # ... and back to the original size after folding (mobilevit_block.py:260-266)
            fm = ops.resize_bilinear(fm, H0, W0)
        fm = self.conv_proj(fm)
        if self.fusion is not None:
            fm = self.fusion(res, x2=fm)  # conv over cat(res, fm) without materialising the cat
        return fm

    def forward_temporal(self, x: Tensor, x_prev: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
        """mobilevit_block.py:289-314: the block of the spatio-temporal MobileViT.  Every TransformerEncoder takes its keys / values from
        `x_prev` — the patches [B*P, N, d] this method returned for the previous frame (None: plain self-attention) — and the patches after
        the last global layer are returned beside the feature map.  Not a path of a §8 model: the patch sequences are materialised in the
        reference's [B*P, N, d] order (torch permutations: plumbing) so that `x_prev` and the returned patches mean what they mean there,
        and the layers run through their [B', S, C] entry points on the same kernels as the spatial path."""
        x = ops.to_nhwc(x)
        res = x
        fm = self.local_rep.conv_1x1(self.local_rep.conv_3x3(x))
        B, d, H, W = fm.shape
        ph, pw = self.patch_h, self.patch_w
        Hn, Wn = int(math.ceil(H / ph) * ph), int(math.ceil(W / pw) * pw)
        interpolate = (Hn != H) or (Wn != W)
        if interpolate:
            fm = ops.resize_bilinear(fm, Hn, Wn)
        n_h, n_w = Hn // ph, Wn // pw
        # unfolding (mobilevit_block.py:185-232): [B, H, W, d] tokens -> [B, p_h, p_w, n_h, n_w, d] -> [B*P, N, d]
        t = ops.tokens_of(fm).reshape(B, n_h, ph, n_w, pw, d)
        patches = t.permute(0, 2, 4, 1, 3, 5).reshape(B * ph * pw, n_h * n_w, d)
        for layer in self.global_rep:
            if isinstance(layer, TransformerEncoder):
                patches = layer(patches, x_prev=x_prev)
            else:
                if not isinstance(layer, nn.LayerNorm):
                    raise NotImplementedError("transformer_norm_layer must be layer_norm on the HIP hot path")
                bp, n, _ = patches.shape
                patches = ops.layer_norm_tokens(patches.reshape(bp * n, d).contiguous(), layer, (bp, n, 1, 1, n, 1, n)).view(bp, n, d)
        # folding (mobilevit_block.py:234-266): back to the [B, H, W, d] token order
        t = patches.view(B, ph, pw, n_h, n_w, d).permute(0, 3, 1, 4, 2, 5).reshape(B * Hn * Wn, d)
        fm = ops.fmap_of(t, B, Hn, Wn)
        if interpolate:
            fm = ops.resize_bilinear(fm, H, W)
        fm = self.conv_proj(fm)
        if self.fusion is not None:
            fm = self.fusion(res, x2=fm)
        return fm, patches

    def forward(self, x: Union[Tensor, Tuple[Tensor]], *args, **kwargs) -> Union[Tensor, Tuple[Tensor, Tensor]]:
        if isinstance(x, Tuple) and len(x) == 2:
            return self.forward_temporal(x=x[0], x_prev=x[1])
        if isinstance(x, Tensor):
            return self.forward_spatial(x)
        raise NotImplementedError


# =============================================================================================
# MobileViTv2  (cvnets/modules/transformer.py:159-264 LinearAttnFFN, cvnets/modules/mobilevit_block.py:329-668 MobileViTBlockv2)
# =============================================================================================
class LinearAttnFFN(nn.Module):
    """pre-norm linear-attention + conv-FFN block.  Runs on the feature map [B, C, H, W]: GroupNorm(1), the 1x1 convs and the
    residuals are position-wise, and the attention kernel addresses the patch groups by stride (see LinearSelfAttention)."""

    def __init__(self, opts, embed_dim: int, ffn_latent_dim: int, attn_dropout: Optional[float] = 0.0, dropout: Optional[float] = 0.1,
                 ffn_dropout: Optional[float] = 0.0, norm_layer: Optional[str] = "layer_norm_2d", *args, **kwargs) -> None:
        super().__init__()
        attn_unit = LinearSelfAttention(opts, embed_dim=embed_dim, attn_dropout=attn_dropout, bias=True)
        self.pre_norm_attn = nn.Sequential(
            get_normalization_layer(opts=opts, norm_type=norm_layer, num_features=embed_dim),
            attn_unit,
            Dropout(p=dropout),
        )
        self.pre_norm_ffn = nn.Sequential(
            get_normalization_layer(opts=opts, norm_type=norm_layer, num_features=embed_dim),
            ConvLayer2d(opts=opts, in_channels=embed_dim, out_channels=ffn_latent_dim, kernel_size=1, stride=1, bias=True, use_norm=False,
                        use_act=True),
            Dropout(p=ffn_dropout),
            ConvLayer2d(opts=opts, in_channels=ffn_latent_dim, out_channels=embed_dim, kernel_size=1, stride=1, bias=True, use_norm=False,
                        use_act=False),
            Dropout(p=dropout),
        )
        self.embed_dim = embed_dim
        self.ffn_dim = ffn_latent_dim
        self.ffn_dropout = ffn_dropout
        self.std_dropout = dropout
        self.attn_fn_name = attn_unit.__repr__()
        self.norm_name = norm_layer

    def __repr__(self) -> str:
        return "{}(embed_dim={}, ffn_dim={}, dropout={}, ffn_dropout={}, attn_fn={}, norm_layer={})".format(
            self.__class__.__name__, self.embed_dim, self.ffn_dim, self.std_dropout, self.ffn_dropout, self.attn_fn_name, self.norm_name)

    def forward(self, x: Tensor, x_prev: Optional[Tensor] = None, patch_hw: Tuple[int, int] = (2, 2), *args, **kwargs) -> Tensor:
        x = ops.to_nhwc(x)
        norm, attn, drop = self.pre_norm_attn[0], self.pre_norm_attn[1], self.pre_norm_attn[2]
        droppy = self.training and drop.p > 0.0
        # x_prev (transformer.py:253-259): the previous frame's feature map, NOT normalised, is the query / key source
        y = attn(norm(x), x_prev=x_prev, patch_hw=patch_hw, residual=None if droppy else x)  # residual rides in out_proj's GEMM epilogue
        x = ops.add(x, drop(y)) if droppy else y
        norm, fc1, drop1, fc2, drop2 = (self.pre_norm_ffn[i] for i in range(5))
        h = drop1(fc1(norm(x)))
        droppy = self.training and drop2.p > 0.0
        y = fc2(h, residual=None if droppy else x)
        return ops.add(x, drop2(y)) if droppy else y


class MobileViTBlockv2(nn.Module):
    """local depthwise 3x3 + 1x1 -> n x LinearAttnFFN + GroupNorm(1) over patch groups -> 1x1 projection (BN)."""

    def __init__(self, opts, in_channels: int, attn_unit_dim: int, ffn_multiplier=2.0, n_attn_blocks: Optional[int] = 2,
                 attn_dropout: Optional[float] = 0.0, dropout: Optional[float] = 0.0, ffn_dropout: Optional[float] = 0.0,
                 patch_h: Optional[int] = 8, patch_w: Optional[int] = 8, conv_ksize: Optional[int] = 3, dilation: Optional[int] = 1,
                 attn_norm_layer: Optional[str] = "layer_norm_2d", *args, **kwargs) -> None:
        super().__init__()
        cnn_out_dim = attn_unit_dim
        conv_3x3_in = ConvLayer2d(opts=opts, in_channels=in_channels, out_channels=in_channels, kernel_size=conv_ksize, stride=1,
                                  use_norm=True, use_act=True, dilation=dilation, groups=in_channels)
        conv_1x1_in = ConvLayer2d(opts=opts, in_channels=in_channels, out_channels=cnn_out_dim, kernel_size=1, stride=1, use_norm=False,
                                  use_act=False)
        self.local_rep = nn.Sequential(conv_3x3_in, conv_1x1_in)
        self.global_rep, attn_unit_dim = self._build_attn_layer(opts=opts, d_model=attn_unit_dim, ffn_mult=ffn_multiplier,
                                                                n_layers=n_attn_blocks, attn_dropout=attn_dropout, dropout=dropout,
                                                                ffn_dropout=ffn_dropout, attn_norm_layer=attn_norm_layer)
        self.conv_proj = ConvLayer2d(opts=opts, in_channels=cnn_out_dim, out_channels=in_channels, kernel_size=1, stride=1, use_norm=True,
                                     use_act=False)
        self.patch_h = patch_h
        self.patch_w = patch_w
        self.patch_area = self.patch_w * self.patch_h
        self.cnn_in_dim = in_channels
        self.cnn_out_dim = cnn_out_dim
        self.transformer_in_dim = attn_unit_dim
        self.dropout = dropout
        self.attn_dropout = attn_dropout
        self.ffn_dropout = ffn_dropout
        self.n_blocks = n_attn_blocks
        self.conv_ksize = conv_ksize
        self.enable_coreml_compatible_fn = opt(opts, "common.enable_coreml_compatible_module", False)
        if self.enable_coreml_compatible_fn:
            raise NotImplementedError("the CoreML-compatible unfolding is an export path, not the HIP hot path")

    def _build_attn_layer(self, opts, d_model: int, ffn_mult, n_layers: int, attn_dropout: float, dropout: float, ffn_dropout: float,
                          attn_norm_layer: str, *args, **kwargs) -> Tuple[nn.Module, int]:
        if isinstance(ffn_mult, (list, tuple)) and len(ffn_mult) == 2:
            step = (ffn_mult[1] - ffn_mult[0]) / max(n_layers - 1, 1)
            ffn_dims = [(ffn_mult[0] + step * i) * d_model for i in range(n_layers)]
        elif isinstance(ffn_mult, (list, tuple)) and len(ffn_mult) == 1:
            ffn_dims = [ffn_mult[0] * d_model] * n_layers
        elif isinstance(ffn_mult, (int, float)):
            ffn_dims = [ffn_mult * d_model] * n_layers
        else:
            raise NotImplementedError
        ffn_dims = [int((d // 16) * 16) for d in ffn_dims]
        global_rep = [LinearAttnFFN(opts=opts, embed_dim=d_model, ffn_latent_dim=ffn_dims[i], attn_dropout=attn_dropout, dropout=dropout,
                                    ffn_dropout=ffn_dropout, norm_layer=attn_norm_layer) for i in range(n_layers)]
        global_rep.append(get_normalization_layer(opts=opts, norm_type=attn_norm_layer, num_features=d_model))
        return nn.Sequential(*global_rep), d_model

    def __repr__(self) -> str:
        s = "{}(".format(self.__class__.__name__) + "\n\t Local representations"
        for m in self.local_rep:
            s += "\n\t\t {}".format(m)
        s += "\n\t Global representations with patch size of {}x{}".format(self.patch_h, self.patch_w)
        for m in self.global_rep:
            s += "\n\t\t {}".format(m)
        s += "\n\t\t {}".format(self.conv_proj)
        return s + "\n)"

    def resize_input_if_needed(self, x: Tensor) -> Tensor:
        B, C, H, W = x.shape
        if H % self.patch_h != 0 or W % self.patch_w != 0:  # mobilevit_block.py:595-603 (align_corners=True)
            nh = int(math.ceil(H / self.patch_h) * self.patch_h)
            nw = int(math.ceil(W / self.patch_w) * self.patch_w)
            x = ops.resize_bilinear(x, nh, nw, align_corners=True)
        return x

    def forward_spatial(self, x: Tensor, *args, **kwargs) -> Tensor:
        x = self.resize_input_if_needed(ops.to_nhwc(x))
        fm = self.local_rep(x)
        phw = (self.patch_h, self.patch_w)
        for layer in self.global_rep:  # F.unfold / F.fold of the reference (:526-555) are index arithmetic inside the attention kernel
            fm = layer(fm, patch_hw=phw) if isinstance(layer, LinearAttnFFN) else layer(fm)
        return self.conv_proj(fm)

    def _fold(self, patches: Tensor, H: int, W: int) -> Tensor:
        """[B, C, P, N] of the reference (F.unfold order: P = i * patch_w + j, N = nh * n_w + nw; mobilevit_block.py:526-540) -> [B, C, H, W]"""
        B, C, P, N = patches.shape
        ph, pw = self.patch_h, self.patch_w
        if P != ph * pw or N != (H // ph) * (W // pw):
            raise NotImplementedError("x_prev must hold the current frame's patch grid ([B, C, patch area, patches])")
        return patches.reshape(B, C, ph, pw, H // ph, W // pw).permute(0, 1, 4, 2, 5, 3).reshape(B, C, H, W)  # plumbing

    def _unfold(self, fm: Tensor) -> Tensor:
        B, C, H, W = fm.shape
        ph, pw = self.patch_h, self.patch_w
        return fm.reshape(B, C, H // ph, ph, W // pw, pw).permute(0, 1, 3, 5, 2, 4).reshape(B, C, ph * pw, (H // ph) * (W // pw))  # plumbing

    def forward_temporal(self, x: Tensor, x_prev: Optional[Tensor], *args, **kwargs) -> Tuple[Tensor, Tensor]:
        """mobilevit_block.py:628-655: every LinearAttnFFN takes its query / key from the previous frame's patches `x_prev` ([B, C, P, N] as
        this method returned them; None: first frame, plain self-attention); returns (feature map, patches after the global layers).  The
        HIP kernels work on the feature map itself, so x_prev is folded once and the returned patches are unfolded once (index
        permutations, torch plumbing)."""
        x = self.resize_input_if_needed(ops.to_nhwc(x))
        fm = self.local_rep(x)
        B, C, H, W = fm.shape
        prev = None
        if x_prev is not None:
            prev = ops.to_nhwc(self._fold(x_prev, H, W).to(fm.dtype))
        phw = (self.patch_h, self.patch_w)
        for layer in self.global_rep:
            fm = layer(fm, x_prev=prev, patch_hw=phw) if isinstance(layer, LinearAttnFFN) else layer(fm)
        return self.conv_proj(fm), self._unfold(fm)

    def forward(self, x, *args, **kwargs):
        if isinstance(x, tuple) and len(x) == 2:
            return self.forward_temporal(x[0], x[1])
        return self.forward_spatial(x)
