"""The convnets of the benchmark configurations, built from plain torch.nn modules, and a small language model of
feed-forward sublayers.

    plain_cnn()              PlainCNN: four conv3x3 (32, 64, 128, 256) + BatchNorm + ReLU + maxpool2x2 blocks in one
                             nn.Sequential (a fused stack), global average pool, linear 256 -> classes
    resnet18()               ResNet-18: 7x7/2 stem + BN + ReLU + 3x3/2 max pool, BasicBlocks [2, 2, 2, 2] at
                             64-128-256-512 channels with 1x1/2 projections, global average pool, linear 512 -> classes
    mobilenet_v3_small()     MobileNetV3-Small-style: inverted residuals with stride-1 depthwise 3x3 / 5x5, 1x1 expand /
                             project, hardswish, BatchNorm, squeeze-excite (adaptive average pool + linear)

    mlp_lm()                 a next-token model without attention: embedding, feed-forward sublayers (ffn.FeedForward) on
                             a residual stream, norm, linear to the vocabulary; serve() gives it with the sublayers'
                             weights in 8 bits

Convolution weights use Kaiming-normal initialization for convolutions (fan-in, ReLU gain), from torch's current RNG state.
These are the model definitions the benchmark configurations name; the reference's own variants differ in input
size, widths and classes (omarchy_mac_torch/models.py in the reference).
"""

import torch
from torch import nn


def _kaiming(model):
    for m in model.modules():
        if isinstance(m, nn.Conv2d):
            nn.init.kaiming_normal_(m.weight, mode="fan_in", nonlinearity="relu")
            if m.bias is not None:
                nn.init.zeros_(m.bias)
    return model


def plain_cnn(classes=10, in_ch=3, widths=(32, 64, 128, 256)):
    layers, c = [], in_ch
    for w in widths:
        layers += [nn.Conv2d(c, w, 3, padding=1, bias=False), nn.BatchNorm2d(w), nn.ReLU(), nn.MaxPool2d(2)]
        c = w
    return _kaiming(nn.Sequential(nn.Sequential(*layers), nn.AdaptiveAvgPool2d(1), nn.Flatten(),
                                  nn.Linear(c, classes)))


class BasicBlock(nn.Module):
    def __init__(self, cin, cout, stride):
        super().__init__()
        self.conv1 = nn.Conv2d(cin, cout, 3, stride, 1, bias=False)
        self.bn1 = nn.BatchNorm2d(cout)
        self.conv2 = nn.Conv2d(cout, cout, 3, 1, 1, bias=False)
        self.bn2 = nn.BatchNorm2d(cout)
        self.relu = nn.ReLU(inplace=True)
        self.down = None
        if stride != 1 or cin != cout:
            self.down = nn.Sequential(nn.Conv2d(cin, cout, 1, stride, bias=False), nn.BatchNorm2d(cout))

    def forward(self, x):
        y = self.relu(self.bn1(self.conv1(x)))
        y = self.bn2(self.conv2(y))
        return self.relu(y + (x if self.down is None else self.down(x)))


class ResNet18(nn.Module):
    def __init__(self, classes=1000, in_ch=3):
        super().__init__()
        self.stem = nn.Sequential(nn.Conv2d(in_ch, 64, 7, 2, 3, bias=False), nn.BatchNorm2d(64), nn.ReLU(inplace=True),
                                  nn.MaxPool2d(3, 2, 1))
        blocks, c = [], 64
        for w, s in ((64, 1), (128, 2), (256, 2), (512, 2)):
            blocks += [BasicBlock(c, w, s), BasicBlock(w, w, 1)]
            c = w
        self.blocks = nn.Sequential(*blocks)
        self.pool = nn.AdaptiveAvgPool2d(1)
        self.fc = nn.Linear(c, classes)
        _kaiming(self)

    def forward(self, x):
        return self.fc(torch.flatten(self.pool(self.blocks(self.stem(x))), 1))


def resnet18(classes=1000):
    return ResNet18(classes)


class SqueezeExcite(nn.Module):
    def __init__(self, c, r=4):
        super().__init__()
        self.pool = nn.AdaptiveAvgPool2d(1)
        self.fc1 = nn.Linear(c, max(8, c // r))
        self.fc2 = nn.Linear(max(8, c // r), c)

    def forward(self, x):
        s = torch.flatten(self.pool(x), 1)
        s = nn.functional.hardsigmoid(self.fc2(nn.functional.relu(self.fc1(s))))
        return x * s[:, :, None, None]


class InvertedResidual(nn.Module):
    def __init__(self, cin, exp, cout, k, se):
        super().__init__()
        self.expand = nn.Sequential(nn.Conv2d(cin, exp, 1, bias=False), nn.BatchNorm2d(exp), nn.Hardswish())
        self.dw = nn.Sequential(nn.Conv2d(exp, exp, k, 1, k // 2, groups=exp, bias=False), nn.BatchNorm2d(exp),
                                nn.Hardswish())
        self.se = SqueezeExcite(exp) if se else nn.Identity()
        self.project = nn.Sequential(nn.Conv2d(exp, cout, 1, bias=False), nn.BatchNorm2d(cout))
        self.residual = cin == cout

    def forward(self, x):
        y = self.project(self.se(self.dw(self.expand(x))))
        return x + y if self.residual else y


class MobileNetV3Small(nn.Module):
    """Stride-1 depthwise convs (the benchmark configuration); resolution drops by 2x2 max pools between stages."""

    def __init__(self, classes=1000, in_ch=3):
        super().__init__()
        self.stem = nn.Sequential(nn.Conv2d(in_ch, 16, 3, 2, 1, bias=False), nn.BatchNorm2d(16), nn.Hardswish())
        cfg = [  # (expansion, out, kernel, squeeze-excite, max pool after)
            (16, 16, 3, True, True), (72, 24, 3, False, True), (88, 24, 3, False, False),
            (96, 40, 5, True, True), (240, 40, 5, True, False), (120, 48, 5, True, False),
            (288, 96, 5, True, True), (576, 96, 5, True, False),
        ]
        layers, c = [], 16
        for exp, out, k, se, pool in cfg:
            layers.append(InvertedResidual(c, exp, out, k, se))
            if pool:
                layers.append(nn.MaxPool2d(2))
            c = out
        self.features = nn.Sequential(*layers)
        self.head = nn.Sequential(nn.Conv2d(c, 576, 1, bias=False), nn.BatchNorm2d(576), nn.Hardswish(),
                                  nn.AdaptiveAvgPool2d(1), nn.Flatten(), nn.Linear(576, classes))
        _kaiming(self)

    def forward(self, x):
        return self.head(self.features(self.stem(x)))


def mobilenet_v3_small(classes=1000):
    return MobileNetV3Small(classes)


class MlpLM(nn.Module):
    """Logits of the next token from the last `context` tokens' embeddings, side by side, through feed-forward sublayers."""

    def __init__(self, vocab, dim, hidden, depth, context=4, act="silu", checkpoint="fp8"):
        from omarchy_mac_torch import ffn  # the operators' library, which a user of the convnets' definitions need not have
        super().__init__()
        if dim % context:
            raise ValueError(f"dim {dim} is not a multiple of the context, {context}")
        self.context = context
        self.embed = nn.Embedding(vocab, dim // context)
        self.blocks = nn.ModuleList(ffn.FeedForward(dim, hidden, act, checkpoint) for _ in range(depth))
        self.norm = ffn.RMSNorm(dim)
        self.head = nn.Linear(dim, vocab, bias=False)
        nn.init.normal_(self.head.weight, std=dim ** -0.5)

    def forward(self, tokens):
        """tokens [batch, length >= context] -> logits [batch, length - context + 1, vocab]"""
        e = self.embed(tokens)
        n = tokens.shape[1] - self.context + 1
        x, stream = torch.cat([e[:, i:i + n] for i in range(self.context)], -1), None
        for block in self.blocks:
            x, stream = block(x, stream)
        y = self.norm(x) if stream is None else self.norm(x, stream)[0]
        return self.head(y)

    def serve(self):
        """A model for inference with the weights of now, its sublayers' in 8 bits: nothing of it is this one's, which stays
        as it is and may train on."""
        import copy
        served = copy.copy(self)
        served._modules = {name: nn.ModuleList(b.serve() for b in m) if name == "blocks" else copy.deepcopy(m)
                           for name, m in self._modules.items()}
        return served.eval().requires_grad_(False)


def mlp_lm(vocab=256, dim=512, hidden=1408, depth=4, **options):
    return MlpLM(vocab, dim, hidden, depth, **options)
