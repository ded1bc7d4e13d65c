"""MultiHeadAttention — mirror of reference utils/attentions.py:44-116 (version 'v2').

Parameter names (linear_k/v/q/final, layer_norm) are the checkpoint contract.  The TTA path only consumes
the attention map (multi_graph_matching.py:498), which comes from csrc/mha.hip without autograd; ``forward`` returns the
(output, attention) pair and is differentiable when gradients are enabled (the source-training loss U_sup.forward
back-propagates through ``output``, multi_graph_matching.py:100-106): the four projections run on the MFMA GEMM
(ops.LinearFn), softmax / LayerNorm are torch glue.  ``attend`` is the layer's output alone, for any number of heads and for batches whose
queries and states are different sets (the reference's forward(key_value_query) with key = value != query)."""
import torch
import torch.nn as nn
import torch.nn.functional as F

from ... import ops


class MultiHeadAttention(nn.Module):
    def __init__(self, model_dim=256, num_heads=4, dropout=0.0, version='v2'):
        super().__init__()
        self.dim_per_head = model_dim // num_heads
        self.num_heads = num_heads
        self.linear_k = nn.Linear(model_dim, self.dim_per_head * num_heads)
        self.linear_v = nn.Linear(model_dim, self.dim_per_head * num_heads)
        self.linear_q = nn.Linear(model_dim, self.dim_per_head * num_heads)
        self.linear_final = nn.Linear(model_dim, model_dim)
        self.dropout = nn.Dropout(dropout)
        self.drop_p = float(dropout)
        self.layer_norm = nn.LayerNorm(model_dim)
        self.version = version
        self._calls = 0

    def attention_only(self, x, seed=None):
        """(n, d) -> (n, n) attention map; no autograd (nothing downstream of it carries gradient on this path)."""
        if self.version != 'v2' or self.num_heads != 1:
            raise NotImplementedError("only the 1-head 'v2' configuration used by MGM3_unsup is implemented")
        with torch.no_grad():
            x = x.detach().contiguous()
            n = x.shape[0]
            q = ops.linear_raw(x, self.linear_q.weight, self.linear_q.bias)
            k = ops.linear_raw(x, self.linear_k.weight, self.linear_k.bias)
            p = self.drop_p if self.training else 0.0
            self._calls += 1
            sd = self._calls if seed is None else seed
            scale = (k.shape[-1] // self.num_heads) ** -0.5            # attentions.py:80
            a = ops.mha_adjacency(q, k, ops.graphs([n]), [n], scale, p, sd, zero_diag=False).view(n, n)
            return a

    def attend(self, query, states, state_lens=None, state_mask=None):
        """layer_norm(query + dropout(linear_final(heads of softmax(q k^T / sqrt(dim_per_head)) v))) without the attention map
        (csrc/attention.hip keeps no map): query (B, n, model_dim), states (B, m, model_dim) or (m, model_dim) for all samples; the states
        j < state_lens[b] with state_mask[b, j] exist (ops.cross_attention).  Dropout acts on the output only, not on the map."""
        if query.dim() != 3 or states.dim() not in (2, 3) or query.shape[2] != self.linear_q.in_features or states.shape[-1] != query.shape[2]:
            raise ValueError("attend: query (B, n, %d) and states (B, m, %d) or (m, %d), got %s and %s" %
                             (self.linear_q.in_features, self.linear_k.in_features, self.linear_k.in_features, tuple(query.shape), tuple(states.shape)))
        B, H, D = query.shape[0], self.num_heads, self.dim_per_head
        if H * D != self.linear_final.in_features:                       # (as in the reference, whose output projection refuses it)
            raise ValueError("attend: %d channels are no %d heads" % (self.linear_final.in_features, H))
        if states.dim() == 3 and states.shape[0] != B:
            raise ValueError("attend: %d samples of queries, %d of states" % (B, states.shape[0]))
        if not query.device == states.device == self.linear_q.weight.device:
            raise ValueError("attend: queries on %s, states on %s, the layer on %s" % (query.device, states.device, self.linear_q.weight.device))
        with ops.on_device_of(query):                                    # (the projections' kernels too, whatever device is current)
            return self._attend(query, states, state_lens, state_mask)

    def _attend(self, query, states, state_lens, state_mask):
        B, H, D = query.shape[0], self.num_heads, self.dim_per_head

        def lin(x, layer):
            if x.numel() == 0:                                           # (the products take no empty operands)
                return F.linear(x.float(), layer.weight, layer.bias)
            y = ops.LinearFn.apply(x.float().reshape(-1, x.shape[-1]).contiguous(), layer.weight, layer.bias)
            return y.view(*x.shape[:-1], layer.out_features)

        def heads(x):
            return x.unflatten(-1, (H, D)) if x.dim() == 3 else x.unflatten(-1, (H, D)).unsqueeze(0).expand(B, -1, -1, -1)

        out = ops.cross_attention(heads(lin(query, self.linear_q)), heads(lin(states, self.linear_k)), heads(lin(states, self.linear_v)),
                                  k_lens=state_lens, key_mask=state_mask)
        return self.layer_norm(query + self.dropout(lin(out.flatten(2), self.linear_final)))

    def forward(self, key_value_query, attn_mask=None):
        key, value, query = key_value_query
        if torch.is_grad_enabled() and (query.requires_grad or self.linear_q.weight.requires_grad):
            if self.version != 'v2' or self.num_heads != 1:
                raise NotImplementedError("only the 1-head 'v2' configuration used by the matching losses is implemented")
            lin = lambda x, l: ops.LinearFn.apply(x.float().contiguous(), l.weight, l.bias)
            k, v, q = lin(key, self.linear_k), lin(value, self.linear_v), lin(query, self.linear_q)
            scale = (k.shape[-1] // self.num_heads) ** -0.5            # attentions.py:80
            attention = self.dropout(torch.softmax((q @ k.t()) * scale, dim=1))   # attentions.py:31-42
            out = self.dropout(lin(attention @ v, self.linear_final))
            return self.layer_norm(query + out).squeeze(), attention.squeeze()
        attention = self.attention_only(query)
        with torch.no_grad():
            v = ops.linear_raw(value.detach().contiguous(), self.linear_v.weight, self.linear_v.bias)
            ctxv = attention @ v
            out = ops.linear_raw(ctxv.contiguous(), self.linear_final.weight, self.linear_final.bias)
            out = self.layer_norm(query.detach() + self.dropout(out))
        return out.squeeze(), attention.squeeze()
