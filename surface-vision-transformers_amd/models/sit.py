"""Surface Vision Transformer on the MI355X-native kernels.

Host-side mirror of the reference's models/sit.py:26-82: same keyword-only constructor, same
attribute names (`to_patch_embedding`, `pos_embedding`, `cls_token`, `dropout`, `transformer`,
`pool`, `to_latent`, `mlp_head` -- the first five are reached from models/mpp.py:115-128), same
state-dict keys (pinned by utils/utils.py:13-33), same forward signature.  The
third-party `vit_pytorch.vit.Transformer` the reference constructs at models/sit.py:57 is
replaced by `Transformer` below, whose parameters keep the PreNorm-generation layout
(layers.i.0.norm / .0.fn.to_qkv / .0.fn.to_out.0 / .1.norm / .1.fn.net.0 / .1.fn.net.3).

All arithmetic runs in libsitk.so (HIP, gfx950).  Additions over the reference API:
  * `compute_dtype` ('bf16' default | 'f16' | 'f32'): MFMA operand type (see include/sitk.h; 'f16' = the mode that meets
    the reference-parity bar of 1e-3 at bf16 speed, backward on a loss-scaled gradient stream; 'f32' = verification mode);
  * forward also accepts a raw channels-last surface (B, 40962, C) and gathers the patches on the
    GPU (tools/preprocessing.py:74-84) with the table registered for (num_patches, num_vertices).
  * `rotary`, `key_blocks`, `act8` (all off by default, for fine patch grids): see Transformer.
There is no CPU forward: tensors must be on the GPU.
"""
import torch
from torch import nn

from .. import functional as Fn
from .. import ops, tables
from ..runtime import SitkError


class PreNorm(nn.Module):
    """Parameter container: LayerNorm(dim) applied before `fn` (keys `.norm.*`, `.fn.*`)."""

    def __init__(self, dim, fn):
        super().__init__()
        self.norm = nn.LayerNorm(dim)
        self.fn = fn


class Attention(nn.Module):
    def __init__(self, dim, heads, dim_head, dropout):
        super().__init__()
        if dim_head > 64 or dim_head < 1:
            raise SitkError(f"dim_head={dim_head}: the attention kernels hold 64 features per head (every reference config uses "
                            "64: config/SiT/training/hparams.yml:33-45); smaller heads run zero-padded, larger ones are not implemented")
        inner = heads * dim_head
        self.heads, self.dim_head = heads, dim_head
        self.scale = dim_head ** -0.5
        self.to_qkv = nn.Linear(dim, inner * 3, bias=False)
        # vit_pytorch: no output projection for a single head as wide as the model
        self.project_out = not (heads == 1 and dim_head == dim)
        self.to_out = nn.Sequential(nn.Linear(inner, dim), nn.Dropout(dropout)) if self.project_out else nn.Identity()


def _capturing(device):
    return torch.device(device).type == "cuda" and torch.cuda.is_current_stream_capturing()


class FeedForward(nn.Module):
    def __init__(self, dim, hidden_dim, dropout):
        super().__init__()
        self.net = nn.Sequential(nn.Linear(dim, hidden_dim), nn.GELU(), nn.Dropout(dropout),
                                 nn.Linear(hidden_dim, dim), nn.Dropout(dropout))


class Transformer(nn.Module):
    """depth x [x += to_out(softmax(q k^T * scale) v); x += W2 gelu(W1 LN(x) + b1) + b2], positional
    ctor (dim, depth, heads, dim_head, mlp_dim, dropout) as at models/sit.py:57.

    Options for fine patch grids; a model with any of them runs stage by stage:
      * rotary: pairs of features per axis, e.g. (10, 10, 12): q and k of every token are turned by its position (set_positions);
        rotary_base: the slowest pair of an axis with n pairs turns by rotary_base^-((n - 1) / n) per unit.
      * key_blocks: (block, top_k): every query attends to the top_k blocks of `block` tokens (a multiple of 64) whose mean key
        it has the largest product with, instead of to all tokens.
      * act8: training keeps the inputs of the linear layers and of GELU in 8 bits (about 29 D instead of 48 D bytes per token and layer
        in the 16-bit modes with mlp_dim = 4 D); forward values are unchanged."""

    rotary, key_blocks, act8, _positions, _positions_captured = None, None, False, None, ()     # also of modules pickled before the options were there

    def __init__(self, dim, depth, heads, dim_head, mlp_dim, dropout=0.0, compute_dtype="bf16", rotary=None, rotary_base=10000.0,
                 key_blocks=None, act8=False):
        super().__init__()
        self.rotary = None if rotary is None else tuple(int(n) for n in rotary)
        if self.rotary is not None and (not 1 <= len(self.rotary) <= 4 or min(self.rotary) < 0
                                        or not 1 <= sum(self.rotary) <= dim_head // 2):
            raise SitkError(f"rotary={rotary}: 1 to 4 axes with 1 to {dim_head // 2} pairs of features together (dim_head={dim_head})")
        if self.rotary is not None and not 0.0 < float(rotary_base) < float("inf"):
            raise SitkError(f"rotary_base={rotary_base}")
        self.rotary_base = float(rotary_base)
        self.key_blocks = None if key_blocks is None else tuple(int(n) for n in key_blocks)
        if self.key_blocks is not None and (len(self.key_blocks) != 2 or self.key_blocks[0] % 64 or not 64 <= self.key_blocks[0] <= 1024
                                            or self.key_blocks[1] < 1):
            raise SitkError(f"key_blocks={key_blocks}: (block, top_k) with a block of 64, 128, ... 1024 tokens and top_k >= 1")
        self.act8 = bool(act8)
        self._positions_dev = {}
        self.dim, self.depth, self.heads, self.mlp_dim = dim, depth, heads, mlp_dim
        self.p_dropout = float(dropout)
        self._drop_state = None
        self.compute_dtype = compute_dtype
        self.layers = nn.ModuleList([
            nn.ModuleList([PreNorm(dim, Attention(dim, heads, dim_head, dropout)),
                           PreNorm(dim, FeedForward(dim, mlp_dim, dropout))])
            for _ in range(depth)])

    def layer_tensors(self):
        """Per layer, the 11 parameters in the C ABI's sitk_layer_params order."""
        out = []
        for attn, ff in self.layers:
            out.append([attn.norm.weight, attn.norm.bias, attn.fn.to_qkv.weight, attn.fn.to_out[0].weight,
                        attn.fn.to_out[0].bias, ff.norm.weight, ff.norm.bias, ff.fn.net[0].weight,
                        ff.fn.net[0].bias, ff.fn.net[3].weight, ff.fn.net[3].bias])
        return out

    def fused_ok(self):
        """The fused per-block kernels cover dropout 0, 64 features per head and a projected attention output -- every
        reference configuration; anything else runs stage by stage."""
        a = self.layers[0][0].fn if len(self.layers) else None
        if self.rotary is not None or self.key_blocks is not None or self.act8:
            return False
        return not (self.training and self.p_dropout > 0) and (a is None or (a.dim_head == 64 and a.project_out))

    def set_positions(self, positions):
        """Positions of the tokens for `rotary`: (N, axes), floating point or integers, one row per token (a class token included).  A captured
        graph keeps the positions that it was captured with."""
        if self.rotary is None:
            raise SitkError("set_positions: the model has no rotary positions (rotary=None)")
        positions = torch.as_tensor(positions).detach()
        if positions.dim() != 2 or positions.shape[1] != len(self.rotary):
            raise SitkError(f"set_positions: ({len(self.rotary)} axes) expected (tokens, {len(self.rotary)}), got {tuple(positions.shape)}")
        if positions.dtype not in (torch.float32, torch.float64, torch.int32, torch.int64):
            positions = positions.to(torch.float32 if positions.is_floating_point() else torch.int64)
        with torch.inference_mode(False):                        # kept beyond the call: a later training step saves them for its backward pass
            self._positions, self._positions_dev = positions.cpu().clone(), {}

    def _rotary_inputs(self, N, device):
        if self._positions is None:
            raise SitkError("rotary positions are not set (SiT.set_patch_positions / Transformer.set_positions)")
        if self._positions.shape[0] != N:
            raise SitkError(f"rotary positions of {self._positions.shape[0]} tokens, the input has {N}")
        key, capturing = str(device), _capturing(device)
        if key not in self._positions_dev:
            if capturing:
                raise SitkError(f"rotary positions are not on {device} yet: run the model once before capturing it")
            with torch.inference_mode(False):
                self._positions_dev[key] = (self._positions.to(device), ops.rope_freqs(self.rotary, self.rotary_base, device))
        inputs = self._positions_dev[key]
        if capturing and not any(inputs is kept for kept in self._positions_captured):
            self._positions_captured = (*self._positions_captured, inputs)     # a replay reads them, whatever set_positions has put in their place
        return inputs

    def _attend(self, qkv, B, N, H, dh, scale):
        """(B, N, 3 H dh) -> (B, N, H dh): rotary positions, then attention over selected blocks or over all tokens."""
        q, k, v = qkv.view(B, N, 3, H, dh).unbind(2)
        if self.rotary is not None:
            q, k = Fn.RopeAxesFn.apply(q, k, *self._rotary_inputs(N, qkv.device), self.rotary)
        if dh != 64:
            q, k, v = (torch.nn.functional.pad(x, (0, 64 - dh)) for x in (q, k, v))
        if self.key_blocks is not None:
            o = Fn.BlockAttentionFn.apply(q, k, v, None, *self.key_blocks, scale, self.compute_dtype)
        else:
            o = Fn.AttentionFn.apply(torch.stack((q, k, v), 2).view(B, N, 3 * H * 64), H, self.compute_dtype, scale).view(B, N, H, 64)
        return o[..., :dh].reshape(B, N, H * dh)

    def _forward_staged(self, x):
        """The block stage by stage -- LayerNorm, Linear, attention, GELU and dropout + residual each as its own libsitk launch
        -- instead of the fused per-block kernels, for what those do not cover: training with dropout > 0 (the three
        nn.Dropout of a vit_pytorch block: behind to_out.0, behind GELU, behind net.3; the fused kernels have no mask
        plumbing), heads narrower than 64 features (q, k, v zero-padded to 64: the scores and the first dim_head output
        features are unchanged) and the projection-free single head.  Every reference configuration sets dropout 0.0 and
        dim_head 64 (config/SiT/training/hparams.yml:33-46): this path exists so that the constructor arguments are honoured,
        not for speed.  The masks come from a device-side Philox stream seeded from torch's seed at first use."""
        dt = self.compute_dtype
        p = self.p_dropout if self.training else 0.0
        if self._drop_state is None or self._drop_state.device != x.device:
            self._drop_state = torch.tensor([torch.initial_seed() & 0x7FFFFFFFFFFFFFFF, 0], dtype=torch.int64, device=x.device)
        st = self._drop_state
        x = x.float()
        B, N, _ = x.shape
        keep8 = self.act8 and torch.is_grad_enabled()
        linear, gelu = (Fn.Linear8Fn, Fn.Gelu8Fn) if keep8 else (Fn.LinearFn, Fn.GeluFn)
        for attn, ff in self.layers:
            a = attn.fn
            H, dh = a.heads, a.dim_head
            h = Fn.LayerNormFn.apply(x, attn.norm.weight, attn.norm.bias)
            qkv = linear.apply(h, a.to_qkv.weight, None, dt)
            if self.rotary is not None or self.key_blocks is not None:
                o = self._attend(qkv, B, N, H, dh, a.scale)
            else:
                if dh != 64:                                       # (h d) per q | k | v: zero features 'dh..63' of every head
                    qkv = torch.nn.functional.pad(qkv.view(B, N, 3 * H, dh), (0, 64 - dh)).view(B, N, 3 * H * 64)
                o = Fn.AttentionFn.apply(qkv, H, dt, a.scale)
                if dh != 64:
                    o = o.view(B, N, H, 64)[..., :dh].reshape(B, N, H * dh)
            y = linear.apply(o, a.to_out[0].weight, a.to_out[0].bias, dt) if a.project_out else o
            x = Fn.DropoutResidualFn.apply(y, x, p, st)
            h = Fn.LayerNormFn.apply(x, ff.norm.weight, ff.norm.bias)
            u = linear.apply(h, ff.fn.net[0].weight, ff.fn.net[0].bias, dt)
            g = gelu.apply(u)
            if p > 0:
                g = Fn.DropoutResidualFn.apply(g, None, p, st)
            y = linear.apply(g, ff.fn.net[3].weight, ff.fn.net[3].bias, dt)
            x = Fn.DropoutResidualFn.apply(y, x, p, st)
        return x

    def forward(self, x):
        if not x.is_cuda:
            raise SitkError("sitk Transformer: input must be on the GPU (no CPU path)")
        if not self.fused_ok():
            return self._forward_staged(x)
        flat = [p for layer in self.layer_tensors() for p in layer]
        cfg = (self.dim, self.depth, self.heads, self.mlp_dim, self.compute_dtype)
        return Fn.EncoderFn.apply(x.float(), cfg, *flat)


class Dropout(nn.Dropout):
    """nn.Dropout(p) of models/sit.py:55 (emb_dropout) on libsitk's Philox stream (same `p` attribute, no parameters);
    identity in eval mode and for p == 0."""

    def __init__(self, p=0.0):
        super().__init__(p)
        self._state = None

    def forward(self, x):
        if not self.training or self.p == 0.0:
            return x
        if not x.is_cuda:
            raise SitkError("sitk Dropout: input must be on the GPU (no CPU path)")
        if self._state is None or self._state.device != x.device:
            self._state = torch.tensor([(torch.initial_seed() + 0x9E3779B9) & 0x7FFFFFFFFFFFFFFF, 0], dtype=torch.int64,
                                       device=x.device)
        return Fn.DropoutResidualFn.apply(x.float(), None, self.p, self._state)


class ToTokens(nn.Module):
    """Index 0 of `to_patch_embedding`: 'b c n v -> b n (v c)' (models/sit.py:49). Returns fp32
    tokens (B, P, V*C) so that external callers (models/mpp.py:82-83 style) see the reference layout."""

    def forward(self, x):
        B, C, P, V = x.shape
        if not x.is_cuda:
            raise SitkError("sitk: input must be on the GPU (no CPU path)")
        K = V * C
        return ops.patchify(x.float(), "f32", ld=ops.pad8(K))[:, :K].reshape(B, P, K)


class PatchLinear(nn.Linear):
    """Index 1 of `to_patch_embedding` (key `to_patch_embedding.1.*`): callable on (B, P, K) fp32
    exactly like the nn.Linear the reference reaches into at models/mpp.py:115."""

    compute_dtype = "bf16"

    def forward(self, x):
        if not x.is_cuda:
            raise SitkError("sitk: input must be on the GPU (no CPU path)")
        return Fn.LinearFn.apply(x.float(), self.weight, self.bias, self.compute_dtype)


class SiT(nn.Module):
    def __init__(self, *, dim, depth, heads, mlp_dim, pool="cls", num_patches=20, num_classes=1, num_channels=4,
                 num_vertices=2145, dim_head=64, dropout=0.0, emb_dropout=0.0, compute_dtype="bf16", rotary=None,
                 rotary_base=10000.0, key_blocks=None, act8=False):
        super().__init__()
        assert pool in {"cls", "mean"}, "pool type must be either cls (cls token) or mean (mean pooling)"
        patch_dim = num_channels * num_vertices
        self.num_patches, self.num_vertices, self.num_channels = num_patches, num_vertices, num_channels
        self.dim, self.patch_dim = dim, patch_dim
        self.compute_dtype = compute_dtype

        self.to_patch_embedding = nn.Sequential(ToTokens(), PatchLinear(patch_dim, dim))
        self.to_patch_embedding[1].compute_dtype = compute_dtype
        self.pos_embedding = nn.Parameter(torch.randn(1, num_patches + 1, dim))
        self.cls_token = nn.Parameter(torch.randn(1, 1, dim))
        self.dropout = Dropout(emb_dropout)
        self.transformer = Transformer(dim, depth, heads, dim_head, mlp_dim, dropout, compute_dtype=compute_dtype,
                                       rotary=rotary, rotary_base=rotary_base, key_blocks=key_blocks, act8=act8)
        self.pool = pool
        self.to_latent = nn.Identity()
        self.mlp_head = nn.Sequential(nn.LayerNorm(dim), nn.Linear(dim, num_classes))
        self._table = None           # numpy (P, V) uint16
        self.allow_synthetic_table = False   # True: the built-in synthetic 1280 x 45 table loads without a warning
        self._table_dev = {}

    # ---- patch table for the raw-surface entry ---------------------------------------------------
    def set_patch_table(self, table_pv):
        """Use a custom (num_patches, num_vertices) table of ico-6 vertex ids."""
        assert tuple(table_pv.shape) == (self.num_patches, self.num_vertices)
        self._table, self._table_dev = table_pv, {}

    def patch_table(self, device):
        if self._table is None:
            self._table = tables.load_table(self.num_patches, self.num_vertices, allow_synthetic=self.allow_synthetic_table)
        key = str(device)
        if key not in self._table_dev:
            self._table_dev[key] = tables.table_tensor(self._table, device)
        return self._table_dev[key]

    # ---- rotary positions ------------------------------------------------------------------------
    def set_patch_positions(self, positions):
        """Positions of the patches for `rotary`: (num_patches, axes), e.g. the patch centres on the unit sphere times a reach.  The
        class token sits at the origin: it is not turned."""
        positions = torch.as_tensor(positions)
        if positions.dim() != 2 or positions.shape[0] != self.num_patches:
            raise SitkError(f"set_patch_positions: expected ({self.num_patches}, axes), got {tuple(positions.shape)}")
        self.transformer.set_positions(torch.cat((torch.zeros_like(positions[:1]), positions)))

    # ---- stages -------------------------------------------------------------------------------------
    def tokens(self, img):
        """(B, C, P, V) pre-patched [reference layout] or (B, 40962, C) raw surface -> (B*P, ld)
        tokens in the compute dtype, zero padded to a multiple of 64 features."""
        if not img.is_cuda:
            raise SitkError("sitk SiT: input must be on the GPU (no CPU path)")
        if img.dim() == 4:
            return ops.patchify(img.float(), self.compute_dtype), img.shape[0]
        if img.dim() == 3:
            if img.shape[1] != tables.ICO6_VERTICES or img.shape[2] != self.num_channels:
                raise SitkError(f"raw surface must be (B, {tables.ICO6_VERTICES}, {self.num_channels}), got {tuple(img.shape)}")
            return ops.gather_tokens(img.float().contiguous(), self.patch_table(img.device), self.compute_dtype), img.shape[0]
        raise SitkError(f"SiT.forward expects (B, C, P, V) or (B, 40962, C), got {tuple(img.shape)}")

    def embed(self, tokens, B):
        lin = self.to_patch_embedding[1]
        x = Fn.EmbedFn.apply(tokens, lin.weight, lin.bias, self.cls_token, self.pos_embedding, B, self.num_patches,
                             self.compute_dtype)
        return self.dropout(x)

    def forward(self, img):
        tokens, B = self.tokens(img)
        x = self.embed(tokens, B)
        x = self.transformer(x)
        ln, fc = self.mlp_head[0], self.mlp_head[1]
        return Fn.HeadFn.apply(self.to_latent(x), ln.weight, ln.bias, fc.weight, fc.bias, self.pool == "mean")
