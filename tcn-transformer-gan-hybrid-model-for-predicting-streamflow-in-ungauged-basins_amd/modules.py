"""nn.Module surfaces of the reference's hot path, backed by the HIP kernels.

Constructor signatures, attribute names and state_dict keys / shapes follow the reference
modules (cited per class) so that its configs, checkpoints and drivers keep working; the
standard torch.nn layers created here are only parameter containers (they are never called),
the arithmetic runs in functional.py's autograd Functions.
"""
from __future__ import annotations

import math
from typing import Dict, List, Optional, Tuple

import torch
import torch.nn as nn

from . import functional as SF
from . import ops


def _need_cuda(t: torch.Tensor, who: str):
    if not t.is_cuda:
        raise RuntimeError(f"{who}: this implementation only runs on an MI355X GPU (got a {t.device} tensor); "
                           "there is no CPU path")


# ------------------------------------------------------------------------------ encoder
class CNNEncoder(nn.Module):
    """Mirror of src/model/cnn_encoder.py:8-97."""

    def __init__(self, input_channels: int, hidden_dim: int, num_layers: int = 2, kernel_size: int = 3,
                 padding: int = 1, use_batchnorm: bool = True):
        super().__init__()
        if kernel_size < 1 or kernel_size > 8 or padding < 0 or padding > 7 or kernel_size - padding > 8:
            raise NotImplementedError("the HIP encoder's gathered GEMM reaches tap offsets -8 .. 7 (forward and transposed): "
                                      "kernel_size 1 to 8, padding 0 to 7, kernel_size - padding at most 8")
        self.input_channels = input_channels
        self.hidden_dim = hidden_dim
        self.num_layers = num_layers
        self.kernel_size, self.padding, self.use_batchnorm = kernel_size, padding, use_batchnorm
        self.target_spatial = 32
        layers: List[nn.Module] = []
        in_ch = input_channels
        for i in range(num_layers):
            out_ch = hidden_dim * (2 ** i)
            layers.append(nn.Conv2d(in_ch, out_ch, kernel_size=kernel_size, padding=padding, bias=not use_batchnorm))
            if use_batchnorm:
                layers.append(nn.BatchNorm2d(out_ch))
            layers.append(nn.ReLU(inplace=True))
            if i < num_layers - 1:
                layers.append(nn.MaxPool2d(kernel_size=2, stride=2))
            in_ch = out_ch
        self.encoder = nn.Sequential(*layers)
        self.out_channels = in_ch
        self.adaptive_pool = nn.AdaptiveAvgPool2d((self.target_spatial, self.target_spatial))

    def _layer_params(self):
        ps = []
        mods = list(self.encoder)
        for i, m in enumerate(mods):
            if isinstance(m, nn.Conv2d):
                if self.use_batchnorm:
                    bn = mods[i + 1]
                    ps += [m.weight, bn.weight, bn.bias, bn.running_mean, bn.running_var]
                else:
                    ps += [m.weight, m.bias]
        return ps

    def forward(self, x: torch.Tensor, nan_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
        """nan_flag (extension, optional): an int32 [1] device tensor that is set to 1 when x holds Inf
        or NaN -- the training loop's input check (src/train.py:193) done by the layout pass."""
        if x.dim() == 5:
            B, T, C, H, W = x.shape
            x = x.reshape(B * T, C, H, W)
        _need_cuda(x, "CNNEncoder")
        if self.training and self.use_batchnorm:      # one multi-tensor launch for all the layers' counters
            torch._foreach_add_([m.num_batches_tracked for m in self.encoder if isinstance(m, nn.BatchNorm2d)], 1)
        if (self.kernel_size, self.padding, self.use_batchnorm) != (3, 1, True):
            # options the model class never passes: gathered-GEMM convs, no specialised kernels
            if nan_flag is not None:
                ops.nan_inf_flag(x.contiguous().float().view(-1), nan_flag)
            return SF.EncoderGeneralFn.apply(x.float(), self.training, SF.compute_dtype(), self.target_spatial,
                                             self.kernel_size, self.padding,
                                             tuple([5 if self.use_batchnorm else 2] * self.num_layers),
                                             *self._layer_params())
        return SF.EncoderFn.apply(x.float(), self.training, SF.compute_dtype(), self.target_spatial, nan_flag,
                                  *self._layer_params())

    def get_output_channels(self) -> int:
        return self.out_channels


# ------------------------------------------------------------------------------ temporal modules
class PositionalEncoding(nn.Module):
    """Mirror of src/model/transformer_module.py:8-38 (buffer `pe` [1, max_len, d_model])."""

    def __init__(self, d_model: int, max_len: int = 5000):
        super().__init__()
        pe = torch.zeros(max_len, d_model)
        position = torch.arange(0, max_len, dtype=torch.float).unsqueeze(1)
        div_term = torch.exp(torch.arange(0, d_model, 2).float() * (-math.log(10000.0) / d_model))
        pe[:, 0::2] = torch.sin(position * div_term)
        if d_model % 2 == 1:
            pe[:, 1::2] = torch.cos(position * div_term[:-1])
        else:
            pe[:, 1::2] = torch.cos(position * div_term)
        self.register_buffer("pe", pe.unsqueeze(0))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _need_cuda(x, "PositionalEncoding")
        return ops.add_pe(x.contiguous().float(), self.pe[0, : x.size(1)].contiguous())


_LAYER_KEYS = ("self_attn.in_proj_weight", "self_attn.in_proj_bias", "self_attn.out_proj.weight",
               "self_attn.out_proj.bias", "linear1.weight", "linear1.bias", "linear2.weight", "linear2.bias",
               "norm1.weight", "norm1.bias", "norm2.weight", "norm2.bias")


def _get_attr(m: nn.Module, dotted: str):
    for part in dotted.split("."):
        m = getattr(m, part)
    return m


class TransformerModule(nn.Module):
    """Mirror of src/model/transformer_module.py:41-124."""

    def __init__(self, input_dim: int, hidden_dim: int, num_layers: int = 2, num_heads: int = 4,
                 dropout: float = 0.2, feedforward_dim: Optional[int] = None):
        super().__init__()
        self.input_dim, self.hidden_dim = input_dim, hidden_dim
        if feedforward_dim is None:
            feedforward_dim = hidden_dim * 4
        self.input_proj = nn.Linear(input_dim, hidden_dim) if input_dim != hidden_dim else None
        self.pos_encoder = PositionalEncoding(hidden_dim, max_len=100)
        layer = nn.TransformerEncoderLayer(d_model=hidden_dim, nhead=num_heads, dim_feedforward=feedforward_dim,
                                           dropout=dropout, batch_first=True, activation="relu")
        self.transformer_encoder = nn.TransformerEncoder(layer, num_layers=num_layers)
        self.num_heads, self.dropout, self.num_layers = num_heads, dropout, num_layers
        self.output_dim = hidden_dim

    def _layer_weights(self):
        ws = []
        for l in self.transformer_encoder.layers:
            ws += [_get_attr(l, k) for k in _LAYER_KEYS]
        return ws

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _need_cuda(x, "TransformerModule")
        B, T, _ = x.shape
        if self.input_proj is not None:
            x = SF.linear(x.reshape(B * T, -1), self.input_proj, SF.compute_dtype()).view(B, T, -1)
        p = self.dropout if self.training else 0.0
        seed = SF.new_seed() if p > 0 else 0
        return SF.TransformerStackFn.apply(x, self.pos_encoder.pe[0], self.num_heads, p, seed,
                                           *self._layer_weights())

    def get_output_dim(self) -> int:
        return self.output_dim


class LSTMModule(nn.Module):
    """Mirror of src/model/lstm_module.py:7-81.  The reference model never enables bidirectional
    (src/model/__init__.py:82-87); the option is built for one layer, where the backward
    direction is the same recurrence over the reversed sequence with its own weights and the
    result is [h_forward, h_backward] (src/model/lstm_module.py:69-73).  Deeper bidirectional
    stacks feed both directions' whole sequences to the next layer, which the kernel (it keeps
    only the last hidden state) does not provide."""

    def __init__(self, input_dim: int, hidden_dim: int, num_layers: int = 1, dropout: float = 0.2,
                 bidirectional: bool = False):
        super().__init__()
        if bidirectional and num_layers != 1:
            raise NotImplementedError("bidirectional LSTM is built for num_layers = 1 only (the reference model never enables it)")
        self.input_dim, self.hidden_dim, self.num_layers, self.bidirectional = input_dim, hidden_dim, num_layers, bool(bidirectional)
        self.input_proj = nn.Linear(input_dim, hidden_dim) if input_dim != hidden_dim else None
        self.lstm = nn.LSTM(input_size=hidden_dim, hidden_size=hidden_dim, num_layers=num_layers,
                            dropout=dropout if num_layers > 1 else 0, bidirectional=self.bidirectional, batch_first=True)
        self.dropout = dropout if num_layers > 1 else 0.0
        self.output_dim = hidden_dim * 2 if self.bidirectional else hidden_dim

    def _weights(self, suffix: str = ""):
        ws = []
        for l in range(self.num_layers):
            ws += [getattr(self.lstm, f"weight_ih_l{l}{suffix}"), getattr(self.lstm, f"weight_hh_l{l}{suffix}"),
                   getattr(self.lstm, f"bias_ih_l{l}{suffix}"), getattr(self.lstm, f"bias_hh_l{l}{suffix}")]
        return ws

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _need_cuda(x, "LSTMModule")
        B, T, _ = x.shape
        if self.input_proj is not None:
            x = SF.linear(x.reshape(B * T, -1), self.input_proj, SF.compute_dtype()).view(B, T, -1)
        p = self.dropout if self.training else 0.0
        seed = SF.new_seed() if p > 0 else 0
        h = SF.LstmFn.apply(x, self.num_layers, p, seed, *self._weights())
        if not self.bidirectional:
            return h
        hb = SF.LstmFn.apply(x.flip(1), 1, 0.0, 0, *self._weights("_reverse"))
        return torch.cat([h, hb], dim=1)

    def get_output_dim(self) -> int:
        return self.output_dim


class LayerNorm(nn.Module):
    """nn.LayerNorm's constructor for one axis, attributes and state_dict keys (the reference holds it inside
    nn.TransformerEncoderLayer, src/model/transformer_module.py:83-91), for rows of any width and
    number.  Called with a second tensor it normalises x + residual and returns (y, x + residual).
    Inside torch.autocast('cuda') rows are taken in bf16 (statistics and weights stay f32)."""

    def __init__(self, normalized_shape: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True):
        super().__init__()
        shape = tuple(normalized_shape) if isinstance(normalized_shape, (tuple, list)) else (int(normalized_shape),)
        if len(shape) != 1:
            raise NotImplementedError("LayerNorm over the last axis only")
        self.normalized_shape, self.eps, self.elementwise_affine = shape, eps, elementwise_affine
        self.weight = nn.Parameter(torch.ones(shape)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(shape)) if elementwise_affine and bias else None

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        _need_cuda(x, "LayerNorm")
        if x.shape[-1:] != self.normalized_shape:
            raise RuntimeError(f"LayerNorm over {self.normalized_shape[0]} values got rows of shape {tuple(x.shape)}")
        if SF.compute_dtype() == torch.bfloat16:
            x = x.to(torch.bfloat16)
        return SF.layer_norm(x, self.weight, self.bias, self.eps, None if residual is None else residual.to(x.dtype))


class DifferentialAttention(nn.Module):
    """Self-attention of [B, T, embed_dim] tokens with the difference of two softmax maps per head, for sequences of
    any length (TransformerModule's fused layers hold at most 8 steps):

        o_h = (softmax(q1 k1^T / sqrt(d)) - lam_h softmax(q2 k2^T / sqrt(d))) v,   d = embed_dim / (2 num_heads)
        lam_h = exp(lambda_q1 . lambda_k1) - exp(lambda_q2 . lambda_k2) + lambda_init  (vectors of d values per head)

    The heads' results go through a LayerNorm over their 2 d values (shared by the heads), are scaled by 1 -
    lambda_init, as is usual to keep their size that of one softmax map's, and projected.  num_kv_heads < num_heads: groups of
    query heads share a key / value head.  `lengths` int32 [B]: tokens of each sample, the others are not attended
    to.  Computes in bf16 inside torch.autocast('cuda'), else in f32; the result is f32 as from the other modules."""

    def __init__(self, embed_dim: int, num_heads: int, num_kv_heads: Optional[int] = None, causal: bool = False,
                 lambda_init: float = 0.8):
        super().__init__()
        kv = num_heads if num_kv_heads is None else num_kv_heads
        if embed_dim % (16 * num_heads) or embed_dim // (2 * num_heads) > 64:
            raise NotImplementedError("DifferentialAttention: embed_dim / (2 num_heads) must be a multiple of 8 up to 64")
        if kv < 1 or num_heads % kv:
            raise ValueError(f"DifferentialAttention: {num_heads} heads cannot share {kv} key / value heads")
        self.embed_dim, self.num_heads, self.num_kv_heads = embed_dim, num_heads, kv
        self.head_dim, self.causal, self.lambda_init = embed_dim // (2 * num_heads), bool(causal), float(lambda_init)
        width = 2 * self.head_dim
        self.in_proj = nn.Linear(embed_dim, (num_heads + 2 * kv) * width)
        self.out_proj = nn.Linear(num_heads * width, embed_dim)
        self.norm = LayerNorm(width)
        for name in ("lambda_q1", "lambda_k1", "lambda_q2", "lambda_k2"):
            self.register_parameter(name, nn.Parameter(0.1 * torch.randn(num_heads, self.head_dim)))

    def lam(self) -> torch.Tensor:
        """The weight of the second map, one per head."""
        return (torch.exp((self.lambda_q1 * self.lambda_k1).sum(-1)) - torch.exp((self.lambda_q2 * self.lambda_k2).sum(-1))
                + self.lambda_init)

    def forward(self, x: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        _need_cuda(x, "DifferentialAttention")
        if x.dim() != 3 or x.shape[-1] != self.embed_dim:
            raise RuntimeError(f"DifferentialAttention: [B, T, {self.embed_dim}] tokens, not {tuple(x.shape)}")
        B, T, _ = x.shape
        if B * T == 0:                  # no token to attend from (a product of no rows is no launch)
            return x.to(torch.float32, copy=True)
        H, kv, d, dt = self.num_heads, self.num_kv_heads, self.head_dim, SF.compute_dtype()
        qkv = SF.linear(x.reshape(B * T, self.embed_dim), self.in_proj, dt).to(dt).view(B, T, -1)
        q, k, v = torch.split(qkv, [H * 2 * d, kv * 2 * d, kv * 2 * d], dim=-1)
        o = SF.diff_attention(q.view(B, T, H, 2, d), k.view(B, T, kv, 2, d), v.view(B, T, kv, 2 * d), self.lam(), self.causal,
                              lengths=lengths)
        o = self.norm(o) * (1.0 - self.lambda_init)
        return SF.linear(o.reshape(B * T, -1), self.out_proj, dt).view(B, T, self.embed_dim)


# ------------------------------------------------------------------------------ decoder
class SimpleUpsamplingDecoder(nn.Module):
    """Mirror of src/model/decoder.py:125-177."""

    def __init__(self, input_channels: int, output_height: int, output_width: int, hidden_channels: int = 64):
        super().__init__()
        self.output_height, self.output_width = output_height, output_width
        self.conv1 = nn.Conv2d(input_channels, hidden_channels, kernel_size=3, padding=1)
        self.relu1 = nn.ReLU(inplace=True)
        self.conv2 = nn.Conv2d(hidden_channels, hidden_channels, kernel_size=3, padding=1)
        self.relu2 = nn.ReLU(inplace=True)
        self.output_conv = nn.Conv2d(hidden_channels, 1, kernel_size=1)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _need_cuda(x, "SimpleUpsamplingDecoder")
        return SF.DecoderFn.apply(x.float(), self.output_height, self.output_width, SF.compute_dtype(),
                                  self.conv1.weight, self.conv1.bias, self.conv2.weight, self.conv2.bias,
                                  self.output_conv.weight, self.output_conv.bias)


# ------------------------------------------------------------------------------ generator
class StreamflowPredictionModel(nn.Module):
    """Mirror of src/model/__init__.py:13-151."""

    def __init__(self, config: Dict):
        super().__init__()
        self.config = config
        model_cfg = config.get("model", {})
        data_cfg = config.get("data", {})
        self.input_channels = model_cfg.get("input_channels", 10)
        self.hidden_dim = model_cfg.get("hidden_dim", 128)
        self.num_layers = model_cfg.get("num_layers", 2)
        self.backbone = model_cfg.get("backbone", "CNN")
        self.temporal_module_type = model_cfg.get("temporal_module", "LSTM")
        self.upscale_factor = data_cfg.get("upscale_factor", 2)
        self.window_size = data_cfg.get("window_size", 5)
        img_size = data_cfg.get("image_size", [128, 128])
        if isinstance(img_size, int):
            self.input_height = self.input_width = int(img_size)
        else:
            self.input_height, self.input_width = int(img_size[0]), int(img_size[1])
        self.output_height = self.input_height * self.upscale_factor
        self.output_width = self.input_width * self.upscale_factor
        if self.hidden_dim % 8:
            raise NotImplementedError("hidden_dim must be a multiple of 8 on the HIP path")
        self.cnn_encoder = CNNEncoder(self.input_channels, self.hidden_dim, self.num_layers, 3, 1, True)
        cnn_out = self.cnn_encoder.get_output_channels()
        enc_h = enc_w = self.cnn_encoder.target_spatial
        feat = cnn_out * enc_h * enc_w
        if self.temporal_module_type.upper() == "TRANSFORMER":
            self.temporal_module = TransformerModule(feat, self.hidden_dim, self.num_layers, num_heads=4, dropout=0.2)
        else:
            self.temporal_module = LSTMModule(feat, self.hidden_dim, self.num_layers, dropout=0.2)
        self.temporal_to_spatial = nn.Linear(self.temporal_module.get_output_dim(), feat)
        self.encoded_h, self.encoded_w, self.cnn_out_channels = enc_h, enc_w, cnn_out
        self.decoder = SimpleUpsamplingDecoder(cnn_out, self.output_height, self.output_width, hidden_channels=64)

    def forward(self, images: torch.Tensor, nan_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
        """nan_flag: see CNNEncoder.forward (an extension; the reference's forward takes images only)."""
        _need_cuda(images, "StreamflowPredictionModel")
        B, T, C, H, W = images.shape
        encoded = self.cnn_encoder(images.reshape(B * T, C, H, W), nan_flag=nan_flag)
        _, oc, he, we = encoded.shape
        t_out = self.temporal_module(encoded.reshape(B, T, -1))
        sp = SF.linear(t_out, self.temporal_to_spatial, SF.compute_dtype())
        return self.decoder(sp.view(B, oc, he, we))

    def forward_windows(self, frames: torch.Tensor, starts: torch.Tensor, window: int) -> torch.Tensor:
        """Eval-mode forward of the windows frames[s : s + window] for s in `starts` (device
        int64 [B]) over frames [N,C,H,W]: every frame is encoded once however many windows share
        it (adjacent evaluation dates share window - 1 of their frames).  Same result as
        forward() on the stacked windows; not available in training mode, where BatchNorm uses
        the statistics of the whole stacked batch."""
        _need_cuda(frames, "StreamflowPredictionModel")
        if self.training:
            raise RuntimeError("forward_windows is an inference path: call model.eval() first")
        N = frames.shape[0]
        B = starts.numel()
        encoded = self.cnn_encoder(frames).float().contiguous()
        _, oc, he, we = encoded.shape
        F = oc * he * we
        rows = (starts.reshape(-1, 1) + torch.arange(window, device=starts.device).reshape(1, -1)).reshape(-1)
        win = torch.empty((B * window, F), device=frames.device, dtype=torch.float32)
        SF.ops.gather_frames(encoded, F, N, rows.contiguous(), F, win)
        t_out = self.temporal_module(win.view(B, window, F))
        sp = SF.linear(t_out, self.temporal_to_spatial, SF.compute_dtype())
        return self.decoder(sp.view(B, oc, he, we))

    def get_num_parameters(self) -> int:
        return sum(p.numel() for p in self.parameters() if p.requires_grad)


# ------------------------------------------------------------------------------ GAN
class PatchDiscriminator(nn.Module):
    """Mirror of src/model/gan.py:7-64."""

    def __init__(self, input_channels: int = 1, hidden_channels: int = 64):
        super().__init__()
        def conv_block(i, o):
            return nn.Sequential(nn.Conv2d(i, o, kernel_size=4, stride=2, padding=1), nn.BatchNorm2d(o),
                                 nn.LeakyReLU(0.2, inplace=True))

        hc = hidden_channels
        self.model = nn.Sequential(
            nn.Conv2d(input_channels, hc, kernel_size=4, stride=2, padding=1),
            nn.LeakyReLU(0.2, inplace=True),
            conv_block(hc, hc * 2), conv_block(hc * 2, hc * 4), conv_block(hc * 4, hc * 8),
            nn.Conv2d(hc * 8, 1, kernel_size=4, stride=1, padding=1))

    def forward(self, x: torch.Tensor, reuse=None, keep_record: bool = False) -> torch.Tensor:
        """Training mode: BatchNorm uses batch statistics and updates its running buffers; eval
        mode: running statistics, no updates (nn.BatchNorm2d semantics; the reference's trainer
        never leaves training mode, src/train.py:213,234-236).
        keep_record: keep this call's activations on `self.last_record` until the next call.
        `reuse`: such a record, taken from an earlier training-mode call on the same input while
        the parameters have not changed -- the forward is then not recomputed (the BatchNorm
        running statistics still advance as for a second call)."""
        _need_cuda(x, "PatchDiscriminator")
        if reuse is not None and not self.training:
            raise RuntimeError("PatchDiscriminator: a forward record can only be reused in training mode")
        m = self.model
        ps = [m[0].weight, m[0].bias]
        for i in (2, 3, 4):
            conv, bn = m[i][0], m[i][1]
            ps += [conv.weight, conv.bias, bn.weight, bn.bias, bn.running_mean, bn.running_var]
        if self.training:      # one multi-tensor launch for the three counters
            torch._foreach_add_([m[i][1].num_batches_tracked for i in (2, 3, 4)], 1)
        ps += [m[5].weight, m[5].bias]
        record = {} if (keep_record and reuse is None) else None
        out = SF.DiscriminatorFn.apply(x.float(), SF.compute_dtype(), self.training, reuse, record, *ps)
        self.last_record = record
        return out

    last_record = None


class _BceWithLogits(nn.Module):
    """nn.BCEWithLogitsLoss() replacement: mean reduction, tensor labels."""

    def forward(self, logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
        _need_cuda(logits, "GANLoss.gan_loss")
        return SF.BceLogitsFn.apply(logits, 0.0, labels.to(logits.device).expand_as(logits))


class _L1(nn.Module):
    def forward(self, a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
        # ImageLoss with nonzero_weight 1 and metric MAE is exactly mean |a - b|
        return ImageLoss(metric="MAE", nonzero_weight=1.0)(a, b)


class GANLoss(nn.Module):
    """Mirror of src/model/gan.py:67-132."""

    def __init__(self, lambda_gan: float = 1.0, lambda_pixel: float = 1.0):
        super().__init__()
        self.lambda_gan, self.lambda_pixel = lambda_gan, lambda_pixel
        self.gan_loss = _BceWithLogits()
        self.pixel_loss = _L1()

    def discriminator_loss(self, disc_real: torch.Tensor, disc_fake: torch.Tensor) -> torch.Tensor:
        _need_cuda(disc_real, "GANLoss.discriminator_loss")
        loss_real = SF.BceLogitsFn.apply(disc_real, 0.9, None)  # label smoothing, src/model/gan.py:102
        loss_fake = SF.BceLogitsFn.apply(disc_fake, 0.0, None)
        return (loss_real + loss_fake) / 2

    def generator_loss(self, disc_fake, generated, target):
        loss_gan = SF.BceLogitsFn.apply(disc_fake, 1.0, None)
        return self.lambda_gan * loss_gan + self.lambda_pixel * self.pixel_loss(generated, target)


# ------------------------------------------------------------------------------ losses
_METRIC = {"MSE": 0, "MAE": 1}


class ImageLoss(nn.Module):
    """Mirror of src/loss.py:9-70."""

    def __init__(self, metric: str = "MSE", upscale_factor: int = 2, nonzero_weight: float = 10.0,
                 zero_threshold: float = 1e-6):
        super().__init__()
        self.metric = metric.upper()
        self.upscale_factor, self.nonzero_weight, self.zero_threshold = upscale_factor, nonzero_weight, zero_threshold
        if self.metric not in _METRIC:
            raise ValueError(f"Unknown metric: {metric}")

    def forward(self, predictions: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        _need_cuda(predictions, "ImageLoss")
        pos, run, offs, S = _no_stations(predictions)
        cfg = (_METRIC[self.metric], float(self.nonzero_weight), float(self.zero_threshold), 1, 0, 1.0, 0.0)
        return SF.ImageStationLossFn.apply(predictions, targets.to(predictions.device), pos, run, offs, 0, cfg)[0]


def _no_stations(pred: torch.Tensor):
    B = pred.shape[0]
    z = torch.zeros(3 + B + 1, device=pred.device, dtype=torch.int32)
    return z[:2].view(-1, 2), z[2:3].view(torch.float32), z[3:], 0


class StationLoss(nn.Module):
    """Mirror of src/loss.py:73-160."""

    def __init__(self, kernel_size: int = 3, metric: str = "MSE"):
        super().__init__()
        self.kernel_size, self.metric = kernel_size, metric.upper()
        if self.metric not in _METRIC:
            raise ValueError(f"Unknown metric: {metric}")

    def forward(self, predictions, station_positions, station_runoffs) -> torch.Tensor:
        _need_cuda(predictions, "StationLoss")
        pos, run, offs, S = SF.pack_stations(station_positions, station_runoffs, predictions.device)
        if S == 0:
            return torch.tensor(0.0, device=predictions.device)  # src/loss.py:157-158: constant, no grad
        # the fused kernel's image term is weighted 0; the target is a same-size placeholder
        cfg = (0, 1.0, 0.0, int(self.kernel_size), _METRIC[self.metric], 0.0, 1.0)
        return SF.ImageStationLossFn.apply(predictions, predictions.detach(), pos, run, offs, S, cfg)[0]


class CombinedLoss(nn.Module):
    """Mirror of src/loss.py:163-236; config keys as src/loss.py:175-194."""

    def __init__(self, config: Dict):
        super().__init__()
        loss_cfg = config.get("loss", {})
        weights = loss_cfg.get("weights", {})
        upscale = config.get("data", {}).get("upscale_factor", 2)
        self.image_weight = weights.get("image", 1.0)
        self.station_weight = weights.get("station", 0.5)
        self.image_loss = ImageLoss(metric=loss_cfg.get("metric", "MSE"), upscale_factor=upscale,
                                    nonzero_weight=float(loss_cfg.get("nonzero_weight", 10.0)),
                                    zero_threshold=float(loss_cfg.get("zero_threshold", 1e-6)))
        scfg = config.get("stations", {})
        self.station_loss = StationLoss(kernel_size=scfg.get("kernel_size", 3), metric=scfg.get("metric", "MSE"))

    def forward(self, predictions, targets, station_positions=None, station_runoffs=None, nan_flag=None
                ) -> Dict[str, torch.Tensor]:
        """nan_flag (not in the reference's signature): an int32 [1] device tensor that is OR-ed with
        1 when the predictions hold Inf / NaN -- the check of src/train.py:198 done by the loss pass,
        which reads every prediction anyway."""
        _need_cuda(predictions, "CombinedLoss")
        if station_positions is not None and station_runoffs is not None:
            pos, run, offs, S = SF.pack_stations(station_positions, station_runoffs, predictions.device)
        else:
            pos, run, offs, S = _no_stations(predictions)
        il, sl = self.image_loss, self.station_loss
        cfg = (_METRIC[il.metric], float(il.nonzero_weight), float(il.zero_threshold), int(sl.kernel_size),
               _METRIC[sl.metric], float(self.image_weight), float(self.station_weight))
        out = SF.ImageStationLossFn.apply(predictions, targets.to(predictions.device), pos, run, offs, S, cfg, nan_flag)
        # `total` carries the gradient of the weighted sum; the two components are reported values
        return {"total": out[0], "image": out[1].detach(), "station": out[2].detach()}
