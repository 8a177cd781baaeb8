"""nn.Conv2d / nn.ConvTranspose2d / nn.Linear with the reference's parameter names
(``weight``, ``bias``) whose compute runs on liblic.

Packed weights ([copad][taps][cpad] in the activation dtype) are cached per
(dtype, geometry) and rebuilt when a parameter is modified in place (its
``_version`` changes) or moved.
"""
from __future__ import annotations

import os
from typing import Optional, Tuple

import torch
import torch.nn as nn

from .. import functional as Fn
from .._ffi import ACT_NONE, ACT_ROUND, EPI_PLAIN, PRO_NONE
from ..functional import Act


# fp32x6 first-conv patch path: opt-in (LIC_PATCHES=1).  It is +0.75 % end to end, but it changes the
# first layer's summation order away from the exact-fp32 kernel's, so near-tie symbols of the timed
# batch flip (5 instead of 0, within the bar) and net_unet_ha_hs B=1 no longer has exactly the exact
# path's flip set (profiles/r03/patch_path_ab.txt)
_PATCHES = os.environ.get("LIC_PATCHES", "0") == "1"


def _param_key(*ps):
    return tuple((p.data_ptr(), p._version) if p is not None else None for p in ps)


class _PackCache:
    def _get_pack(self, key, build):
        cache = self.__dict__.setdefault("_lic_packs", {})
        ent = cache.get(key)
        pk = _param_key(self.weight, self.bias)
        if ent is None or ent[0] != pk:
            ent = (pk, build())
            cache[key] = ent
        return ent[1]


class Conv2d(nn.Conv2d, _PackCache):
    """nn.Conv2d (square kernel, symmetric padding) executed by lic_conv2d_fwd."""

    def packed(self, dtype: torch.dtype, pad: Optional[Tuple[int, int, int, int]] = None,
               cin_to: Optional[int] = None, cpad_to: Optional[int] = None) -> Fn.ConvPack:
        if pad is None:
            p = self.padding[0]
            pad = (p, p, p, p)
        return self._get_pack((dtype, pad, cin_to, cpad_to), lambda: Fn.pack_conv2d(
            self.weight, self.bias, self.stride[0], pad, dtype, self.groups, cin_to, cpad_to))

    def run(self, x: Act, out: Optional[Act] = None, *, pad=None, act: int = ACT_NONE, slope: float = 0.01,
            epi: int = EPI_PLAIN, r1: Optional[Act] = None, g: Optional[Act] = None, r2: Optional[Act] = None,
            y2: Optional[Act] = None, prologue: int = PRO_NONE, shuffle: bool = False) -> Act:
        k = self.kernel_size[0]
        square = (self.kernel_size[0] == self.kernel_size[1] and self.stride[0] == self.stride[1] and
                  (pad is not None or self.padding[0] == self.padding[1]) and self.dilation == (1, 1))
        if (Fn.split_mode() == 2 and x.dtype == torch.float32 and self.groups == 1 and x.c == self.in_channels and
                x.c <= 4 and 1 < k * k * x.c <= 32 and prologue == PRO_NONE and not shuffle and _PATCHES and square):
            # fp32x6, the image's k x k conv (Cin 3): one 1x1 launch over the patch map (K = 27 -> 32)
            # instead of k*k taps of a 16-channel-padded input on the exact-fp32 kernel (square kernel,
            # stride and padding only: the patch packer takes one of each)
            if pad is None:
                p = self.padding[0]
                pad = (p, p, p, p)
            pk, dy, dx, s = self._get_pack((x.dtype, pad, "patches", x.c), lambda: Fn.pack_conv2d_patches(
                self.weight, self.bias, self.stride[0], pad, x.c, x.dtype))
            Ho, Wo = Fn.conv_out_hw(x.H, x.W, Fn.ConvPack(w=pk.w, bias=None, ci=x.c, co=self.out_channels,
                                                        dy=dy, dx=dx, stride=s, pad=pad, kh=k, kw=k))
            pm = Fn.patches(x, dy, dx, s, Ho, Wo, pk.cpad)
            return Fn.conv(pm, pk, out, act=act, slope=slope, epi=epi, r1=r1, g=g, r2=r2, y2=y2)
        epc = 16 // x.t.element_size()
        if self.groups == 1 and x.c % epc and x.zpad >= -(-x.c // epc) * epc and x.c == self.in_channels:
            # zero-padded small-channel input (e.g. the 3-channel image): run as Cin = 16 B on MFMA
            cp = -(-x.c // epc) * epc
            # fp32 (the image's 3 channels, exact-fp32 halo kernel): ONE 8-channel chunk instead of the
            # 16 the packs default to -- the second chunk was all zeros on both sides, so the result is
            # bit-identical at half the MFMA work
            # (k x k only: the 1x1 skip keeps its 16-channel pack and kernels)
            cpad8 = 8 if (x.dtype == torch.float32 and cp <= 8 and k > 1) else None
            pk = self.packed(x.dtype, pad, cin_to=cp, cpad_to=cpad8)
            return Fn.conv(Act(x.t, x.c0, cp), pk, out, act=act, slope=slope, epi=epi, r1=r1, g=g, r2=r2, y2=y2,
                           prologue=prologue, shuffle=shuffle)
        pk = self.packed(x.dtype, pad)
        return Fn.conv(x, pk, out, act=act, slope=slope, epi=epi, r1=r1, g=g, r2=r2, y2=y2, prologue=prologue,
                       shuffle=shuffle)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.run(Act.from_nchw(x)).nchw()


class Linear(nn.Linear, _PackCache):
    """nn.Linear applied per pixel of an NHWC map (a 1x1 convolution).  ``int8``: whether functional.int8_linears takes
    this layer (the window-attention blocks' qkv and proj are taken)."""

    int8 = False

    def packed(self, dtype: torch.dtype) -> Fn.ConvPack:
        return self._get_pack(dtype, lambda: Fn.pack_conv2d(self.weight[:, :, None, None], self.bias, 1,
                                                             (0, 0, 0, 0), dtype))

    def packed_int8(self) -> Fn.Int8Pack:
        return self._get_pack("int8", lambda: Fn.pack_linear_int8(self.weight, self.bias))

    def run(self, x: Act, out: Optional[Act] = None, **kw) -> Act:
        """Inside functional.int8_linears the product of a layer with ``int8`` runs in 8-bit integers, for the epilogues
        linear_int8 has (activation and residual); other calls keep the activation dtype's products."""
        if self.int8 and Fn.int8_mode() and kw.keys() <= {"act", "slope", "r1"} and kw.get("act", ACT_NONE) != ACT_ROUND:
            return Fn.linear_int8(x, self.packed_int8(), out, **kw)
        return Fn.conv(x, self.packed(x.dtype), out, **kw)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        shp = x.shape
        t = x.reshape(-1, 1, 1, shp[-1]).contiguous()
        out = self.run(Act(t))
        return out.t.reshape(*shp[:-1], self.out_features)


class ConvTranspose2d(nn.ConvTranspose2d, _PackCache):
    """nn.ConvTranspose2d as stride^2 sub-pixel phase convolutions (gather form),
    optionally preceded by ZeroPad2d(left=prepad[1], top=prepad[0])."""

    def packed(self, dtype: torch.dtype, prepad=(0, 0)):
        return self._get_pack((dtype, prepad), lambda: Fn.pack_conv_transpose2d(
            self.weight, self.bias, self.stride[0], self.padding[0], self.output_padding[0], dtype, prepad))

    def packed_fused(self, dtype: torch.dtype, prepad=(0, 0)):
        """All four phases in one launch (out_shuffle=3), or None (see pack_conv_transpose2d_fused)."""
        return self._get_pack((dtype, prepad, "fused"), lambda: Fn.pack_conv_transpose2d_fused(
            self.weight, self.bias, self.stride[0], self.padding[0], dtype, prepad))

    def out_hw(self, H, W, prepad=(0, 0)):
        return Fn.convT_out_hw(H, W, self.stride[0], self.padding[0], self.output_padding[0], self.kernel_size[0],
                               prepad)

    # narrow stride-2 layers (s_model's 192 -> 16 output layer) run as one fused launch:
    # 4 phases x co channels fill a 64-wide MFMA tile instead of four half-empty ones
    FUSED_MAX_CO = 16

    def run(self, x: Act, out: Optional[Act] = None, *, prepad=(0, 0), **kw) -> Act:
        Ho, Wo = self.out_hw(x.H, x.W, prepad)
        if (self.stride[0] == 2 and self.out_channels <= self.FUSED_MAX_CO and Ho % 2 == 0 and Wo % 2 == 0
                and not kw):
            fpk = self.packed_fused(x.dtype, prepad)
            if fpk is not None:
                if out is None:
                    out = Act.empty(x.B, Ho, Wo, self.out_channels, x.dtype, x.t.device)
                return Fn.conv(x, fpk, out, out_hw=(Ho // 2, Wo // 2), shuffle=3)
        packs = self.packed(x.dtype, prepad)
        if self.stride[0] == 1 and self.kernel_size[0] == 1 and self.padding[0] == 0:
            # 1x1 stride-1 transposed conv == 1x1 conv with the transposed weight (one phase).
            return Fn.conv(x, packs[0], out if out is not None else Act.empty(x.B, Ho, Wo, packs[0].co, x.dtype,
                                                                               x.t.device), **kw)
        return Fn.conv_transpose(x, packs, Ho, Wo, out, **kw)

    def forward(self, x: torch.Tensor, output_size=None) -> torch.Tensor:
        return self.run(Act.from_nchw(x)).nchw()
