"""torch.nn layers over the fused GPU ops: the user-facing counterpart of the reference's
`haste_pytorch` package (frameworks/pytorch/{lstm,gru,indrnn,layer_norm_lstm,layer_norm_gru,
layer_norm_indrnn,base_rnn}.py) with the same class names, constructor arguments, parameter
names, shapes, gate orders and initialisers, the same `forward(input, state=None,
lengths=None)` contract and the same `to_native_weights` / `from_native_weights` maps.

As in the reference (frameworks/pytorch/lstm.py:244-266, base_rnn.py:72-76), `_is_cuda()`
decides per call between the fused GPU op and a plain torch loop over the time steps written
here (`_eager_*`): layers whose parameters live on the CPU run that loop, and patching
`_is_cuda` to return False (what the reference's validation/pytorch.py:42-62 does to compare
its two paths) runs it on GPU tensors too.  The loop is differentiated by autograd and is
never taken for GPU parameters unless patched in.

Differences, on purpose:
  * DropConnect of LSTM and GRU is applied inside the recurrence kernel while it loads the
    recurrent matrix (the mask is drawn here and handed over), instead of materialising a
    dropped-out copy of the matrix first (frameworks/pytorch/lstm.py:252).

CausalConv, SelectiveScan and ResidualNorm, at the end, are the layers of a state space block; the reference has
none of them.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops

__all__ = ["LSTM", "GRU", "IndRNN", "LayerNormLSTM", "LayerNormGRU", "LayerNormIndRNN",
           "CausalConv", "SelectiveScan", "ResidualNorm"]


def _t(w):
    return ops.transpose(w) if w.is_cuda and w.is_contiguous() else w.t().contiguous()


def _single_shot(ctx, name):
    """The fused backward passes overwrite the activations the forward pass saved (as the
    reference's do, lib/lstm_backward_gpu.cu.cc:92-95), so a graph can be walked once."""
    if getattr(ctx, "consumed", False):
        raise RuntimeError("%s: backward through the same forward pass twice is not supported "
                           "(the saved activations were consumed by the first)" % name)
    ctx.consumed = True


def _no_training_backward(name):
    return RuntimeError("%s backward can only be called in training mode" % name)


# ---- autograd glue (reference frameworks/pytorch/lstm.py:69-88 and siblings) -------------
# The functions return what the layers return -- the states after each step and what `wanted` asks for
# of every state -- and not the [T+1,N,H] sequences the ops work on: differentiating slices of those
# would fill and copy a sequence per slice, where the backward ops take the gradients of the outputs
# as they come (a training step of the IndRNN at T=2500 N=64 H=4096, 2.6 GB per sequence: 10.0 -> 8.7 ms;
# of the LSTM at N=128 T=100 C=H=512 1399 -> 1367 us).
def _alias(seq, first):
    """seq[first:] (or seq[-1]) as a tensor on the same memory that is no view to autograd."""
    a = seq[first:] if first >= 0 else seq[-1]
    return seq.new_empty(0).set_(a)


def _one_per_row(wanted, seq):
    """Whether an index tensor is what the ops take: a step for every batch row (anything else that
    indexing accepts is left to it)."""
    return wanted.dim() == 1 and wanted.size(0) == seq.size(1) and wanted.is_contiguous() and seq.numel() > 0


# Outputs that share memory must share a version counter, or autograd does not see that a change of one
# (padding masked in place, say) changes another that was saved: the states of h that y holds are either
# views of y, taken by the layer (None here), or a copy (3 us) where a view would bring back the gradients
# of slices.
def _wanted_states(seqs, wanted):
    """What a layer returns of its state sequences [T+1,N,H], h's first: "last" [N,H] ("last of y" where
    nothing is differentiated), "all" [T,N,H], or the states at the steps in an index tensor [N].  None:
    the layer takes it from y."""
    if torch.is_tensor(wanted):
        if _one_per_row(wanted, seqs[0]):
            return ops.gather_states(seqs, wanted)
        cols = torch.arange(seqs[0].size(1), device=wanted.device)
        return tuple(seq[wanted, cols] for seq in seqs)
    h = seqs[0][-1].clone() if wanted == "last" else None
    return (h,) + tuple(_alias(seq, 1 if wanted == "all" else -1) for seq in seqs[1:])


def _upstream(like, grad_steps, grad_wanted, wanted):
    """The gradients of a state sequence `like` [T+1,N,H] from those of the states after each step and of
    the wanted states (either may be None): (gradients [T,N,H] or [T+1,N,H], or None; more of the last
    states, [N,H] or None)."""
    if grad_wanted is None:
        return grad_steps if grad_steps is None else grad_steps.contiguous(), None
    if not torch.is_tensor(wanted):
        if wanted == "last":
            return grad_steps if grad_steps is None else grad_steps.contiguous(), grad_wanted
        return grad_wanted.contiguous(), None  # of c: those of h are y's
    if _one_per_row(wanted, like):
        return ops.state_gradients(like, grad_steps, grad_wanted, wanted), None
    full = torch.zeros_like(like) if grad_steps is None else torch.empty_like(like)
    if grad_steps is not None:
        full[1:] = grad_steps
        full[0].zero_()
    cols = torch.arange(like.size(1), device=like.device)
    # several steps of a row may be asked for, the same one twice among them
    full.index_put_((wanted, cols), grad_wanted, accumulate=True)
    return full, None


def _upstream_h(h, grad_y, grad_h, wanted):
    grad, last = _upstream(h, grad_y, grad_h, wanted)
    return h.new_zeros((h.size(0) - 1,) + h.shape[1:]) if grad is None else grad, last


def _initial(ctx, *grads):
    """The gradients of the initial states, inputs 4, 5 of every function, where they are tensors."""
    return tuple(g if ctx.needs_input_grad[4 + i] else None for i, g in enumerate(grads))


class _RecurrenceFunction(torch.autograd.Function):
    """forward(ctx, training, zoneout_prob, wanted, ...) -> the outputs named above; the subclasses call
    the ops."""

    @staticmethod
    def finish(ctx, training, wanted, saved, *seqs):
        """Saves what the backward pass needs; (y, wanted states of each sequence)."""
        h = seqs[0]
        y = _alias(h, 1)
        states = _wanted_states(seqs, wanted)
        # the outputs that share memory with h and c too: if a caller changes them, autograd notices
        ctx.save_for_backward(y, *states, *saved)
        if torch.is_tensor(wanted):  # often the caller's own tensor, filled again for the next batch
            wanted = wanted.clone() if wanted.is_inference() else wanted
            ctx.lengths_version = None if wanted.is_inference() else wanted._version  # None: in inference mode
        ctx.training, ctx.wanted, ctx.count = training, wanted, len(seqs)
        ctx.set_materialize_grads(False)
        return (y,) + states

    @staticmethod
    def restore(ctx, *state_grads):
        """The saved tensors.  Gradients of states at lengths need the lengths of the forward pass (which
        are not saved with the rest: a pass that only y's gradients enter may outlive them)."""
        if (torch.is_tensor(ctx.wanted) and ctx.wanted._version != ctx.lengths_version
                and any(g is not None for g in state_grads)):
            raise RuntimeError("the lengths needed for gradient computation have been modified by an inplace "
                               "operation since the forward pass")
        return ctx.saved_tensors[1 + ctx.count:]


class _LSTMFunction(_RecurrenceFunction):
    @staticmethod
    def forward(ctx, training, zoneout_prob, wanted, x, h0, c0, kernel, recurrent_kernel, bias, zoneout_mask,
                dropconnect_mask, dropconnect_scale):
        h, c, cache = ops.lstm_forward(training, zoneout_prob, x, h0, c0, kernel, recurrent_kernel,
                                       bias, zoneout_mask, dropconnect_mask, dropconnect_scale)
        ctx.dropconnect_scale = dropconnect_scale
        return _RecurrenceFunction.finish(
            ctx, training, wanted,
            (x, kernel, recurrent_kernel, bias, zoneout_mask, h, c, cache, dropconnect_mask), h, c)

    @staticmethod
    def backward(ctx, grad_y, grad_h, grad_c):
        if not ctx.training:
            raise _no_training_backward("LSTM")
        x, kernel, recurrent_kernel, bias, zoneout_mask, h, c, cache, dmask = _RecurrenceFunction.restore(ctx, grad_h, grad_c)
        if dmask is not None:
            recurrent_kernel = recurrent_kernel * dmask * ctx.dropconnect_scale
        _single_shot(ctx, "LSTM")  # the backward pass overwrites the activation cache
        dh_new, dh_last = _upstream_h(h, grad_y, grad_h, ctx.wanted)
        dc_new, dc_last = _upstream(c, None, grad_c, ctx.wanted)
        dx, dh, dc, dW, dR, db = ops.lstm_backward(
            *ops.transpose3(x, kernel, recurrent_kernel), bias, zoneout_mask, h, c, cache, dh_new, dc_new,
            dh_last, dc_last)
        if dmask is not None:
            dR = dR * dmask * ctx.dropconnect_scale
        return (None, None, None, dx) + _initial(ctx, dh, dc) + (dW, dR, db, None, None, None)


class _GRUFunction(_RecurrenceFunction):
    @staticmethod
    def forward(ctx, training, zoneout_prob, wanted, x, h0, kernel, recurrent_kernel, bias, recurrent_bias,
                zoneout_mask, dropconnect_mask, dropconnect_scale):
        h, cache = ops.gru_forward(training, zoneout_prob, x, h0, kernel, recurrent_kernel, bias,
                                   recurrent_bias, zoneout_mask, dropconnect_mask, dropconnect_scale)
        ctx.dropconnect_scale = dropconnect_scale
        return _RecurrenceFunction.finish(
            ctx, training, wanted,
            (x, kernel, recurrent_kernel, bias, recurrent_bias, zoneout_mask, h, cache, dropconnect_mask), h)

    @staticmethod
    def backward(ctx, grad_y, grad_h):
        if not ctx.training:
            raise _no_training_backward("GRU")
        (x, kernel, recurrent_kernel, bias, recurrent_bias, zoneout_mask, h, cache,
         dmask) = _RecurrenceFunction.restore(ctx, grad_h)
        if dmask is not None:
            recurrent_kernel = recurrent_kernel * dmask * ctx.dropconnect_scale
        dh_new, dh_last = _upstream_h(h, grad_y, grad_h, ctx.wanted)
        dx, dh, dW, dR, dbx, dbr = ops.gru_backward(
            *ops.transpose3(x, kernel, recurrent_kernel), bias, recurrent_bias, zoneout_mask, h, cache, dh_new,
            dh_last)
        if dmask is not None:
            dR = dR * dmask * ctx.dropconnect_scale
        return (None, None, None, dx) + _initial(ctx, dh) + (dW, dR, dbx, dbr, None, None, None)


class _IndRNNFunction(_RecurrenceFunction):
    @staticmethod
    def forward(ctx, training, zoneout_prob, wanted, x, h0, kernel, recurrent_scale, bias, zoneout_mask):
        h = ops.indrnn_forward(training, zoneout_prob, x, h0, kernel, recurrent_scale, bias, zoneout_mask)
        return _RecurrenceFunction.finish(ctx, training, wanted,
                                          (x, kernel, recurrent_scale, bias, zoneout_mask, h), h)

    @staticmethod
    def backward(ctx, grad_y, grad_h):
        if not ctx.training:
            raise _no_training_backward("IndRNN")
        x, kernel, recurrent_scale, bias, zoneout_mask, h = _RecurrenceFunction.restore(ctx, grad_h)
        dh_new, dh_last = _upstream_h(h, grad_y, grad_h, ctx.wanted)
        dx, dh, dW, du, db = ops.indrnn_backward(ops.transpose(x), ops.transpose(kernel), recurrent_scale, bias,
                                                 zoneout_mask, h, dh_new, dh_last)
        return (None, None, None, dx) + _initial(ctx, dh) + (dW, du, db, None)


class _LayerNormIndRNNFunction(_RecurrenceFunction):
    @staticmethod
    def forward(ctx, training, zoneout_prob, wanted, x, h0, kernel, recurrent_scale, bias, gamma, zoneout_mask):
        h, act_Wx, cache = ops.layer_norm_indrnn_forward(training, zoneout_prob, x, h0, kernel,
                                                         recurrent_scale, bias, gamma, zoneout_mask)
        return _RecurrenceFunction.finish(
            ctx, training, wanted, (x, kernel, recurrent_scale, bias, gamma, zoneout_mask, h, act_Wx, cache), h)

    @staticmethod
    def backward(ctx, grad_y, grad_h):
        if not ctx.training:
            raise _no_training_backward("LayerNormIndRNN")
        (x, kernel, recurrent_scale, bias, gamma, zoneout_mask, h, act_Wx,
         cache) = _RecurrenceFunction.restore(ctx, grad_h)
        dh_new, dh_last = _upstream_h(h, grad_y, grad_h, ctx.wanted)
        dx, dh, dW, du, db, dgamma = ops.layer_norm_indrnn_backward(
            ops.transpose(x), ops.transpose(kernel), recurrent_scale, bias, gamma, zoneout_mask, h, act_Wx, cache,
            dh_new, dh_last)
        return (None, None, None, dx) + _initial(ctx, dh) + (dW, du, db, dgamma, None)


class _LayerNormLSTMFunction(_RecurrenceFunction):
    @staticmethod
    def forward(ctx, training, zoneout_prob, wanted, x, h0, c0, kernel, recurrent_kernel, bias, gamma, gamma_h,
                beta_h, zoneout_mask):
        outs = ops.layer_norm_lstm_forward(training, zoneout_prob, x, h0, c0, kernel, recurrent_kernel,
                                           bias, gamma, gamma_h, beta_h, zoneout_mask)
        return _RecurrenceFunction.finish(
            ctx, training, wanted,
            (x, kernel, recurrent_kernel, bias, gamma, gamma_h, beta_h, zoneout_mask) + tuple(outs), *outs[:2])

    @staticmethod
    def backward(ctx, grad_y, grad_h, grad_c):
        if not ctx.training:
            raise _no_training_backward("LayerNormLSTM")
        (x, kernel, recurrent_kernel, bias, gamma, gamma_h, beta_h, zoneout_mask, h, c, act_Wx,
         act_Wx_norm, cache1, act_Rh, cache2, act_c_norm, cache3) = _RecurrenceFunction.restore(ctx, grad_h, grad_c)
        _single_shot(ctx, "LayerNormLSTM")  # the saved activations are overwritten below
        dh_new, dh_last = _upstream_h(h, grad_y, grad_h, ctx.wanted)
        dc_new, dc_last = _upstream(c, None, grad_c, ctx.wanted)
        dx, dh, dc, *grads = ops.layer_norm_lstm_backward(
            *ops.transpose3(x, kernel, recurrent_kernel), bias, gamma, gamma_h, beta_h,
            zoneout_mask, h, c, act_Wx, act_Wx_norm, cache1, act_Rh, cache2, act_c_norm, cache3,
            dh_new, dc_new, dh_last, dc_last)
        return (None, None, None, dx) + _initial(ctx, dh, dc) + tuple(grads) + (None,)


class _LayerNormGRUFunction(_RecurrenceFunction):
    @staticmethod
    def forward(ctx, training, zoneout_prob, wanted, x, h0, kernel, recurrent_kernel, bias, recurrent_bias,
                gamma, zoneout_mask):
        outs = ops.layer_norm_gru_forward(training, zoneout_prob, x, h0, kernel, recurrent_kernel, bias,
                                          recurrent_bias, gamma, zoneout_mask)
        return _RecurrenceFunction.finish(
            ctx, training, wanted,
            (x, kernel, recurrent_kernel, bias, recurrent_bias, gamma, zoneout_mask) + tuple(outs), outs[0])

    @staticmethod
    def backward(ctx, grad_y, grad_h):
        if not ctx.training:
            raise _no_training_backward("LayerNormGRU")
        (x, kernel, recurrent_kernel, bias, recurrent_bias, gamma, zoneout_mask, h, cache, act_Wx,
         cache1, act_Rh, cache2) = _RecurrenceFunction.restore(ctx, grad_h)
        dh_new, dh_last = _upstream_h(h, grad_y, grad_h, ctx.wanted)
        dx, dh, *grads = ops.layer_norm_gru_backward(
            *ops.transpose3(x, kernel, recurrent_kernel), bias, recurrent_bias, gamma,
            zoneout_mask, h, cache, act_Wx, cache1, act_Rh, cache2, dh_new, dh_last)
        return (None, None, None, dx) + _initial(ctx, dh) + tuple(grads) + (None,)


# ---- the time loop in plain torch (reference *Script functions, e.g. frameworks/pytorch/
# lstm.py:33-66, gru.py:33-66, layer_norm_lstm.py:31-66, layer_norm_gru.py:31-64,
# indrnn.py:32-51, layer_norm_indrnn.py:32-53) -------------------------------------------------
def _eager_recurrence(step, first, steps, training, zoneout_prob, zoneout_mask):
    """Runs `step(t, states) -> states` for t = 0 .. steps-1 from the states `first` (a tuple,
    hidden state first) and returns each state's sequence stacked to [steps+1, N, H].  Zoneout
    acts on the hidden state only: the mask picks new or old during training, inference blends
    (reference frameworks/pytorch/lstm.py:58-62)."""
    history = [[s] for s in first]
    for t in range(steps):
        new = list(step(t, tuple(seq[-1] for seq in history)))
        if zoneout_prob:
            old_h = history[0][-1]
            if training:
                new[0] = (new[0] - old_h) * zoneout_mask[t] + old_h
            else:
                new[0] = zoneout_prob * old_h + (1 - zoneout_prob) * new[0]
        for seq, value in zip(history, new):
            seq.append(value)
    return tuple(torch.stack(seq) for seq in history)


def _norm(v, gamma, beta=None):
    return F.layer_norm(v, (v.shape[-1],), weight=gamma, bias=beta)


def _eager_lstm(training, zoneout_prob, x, h0, c0, kernel, recurrent_kernel, bias, zoneout_mask,
                gamma=None, gamma_h=None, beta_h=None):
    """LSTM (gamma None) or LayerNormLSTM: returns (h, c), each [T+1, N, H]."""
    wx = x @ kernel if gamma is None else _norm(x @ kernel, gamma[0])

    def step(t, state):
        h, c = state
        rh = h @ recurrent_kernel if gamma is None else _norm(h @ recurrent_kernel, gamma[1])
        i, g, f, o = torch.chunk(rh + wx[t] + bias, 4, dim=1)
        c_new = torch.sigmoid(f) * c + torch.sigmoid(i) * torch.tanh(g)
        seen = c_new if gamma is None else _norm(c_new, gamma_h, beta_h)
        return torch.sigmoid(o) * torch.tanh(seen), c_new

    return _eager_recurrence(step, (h0, c0), x.shape[0], training, zoneout_prob, zoneout_mask)


def _eager_gru(training, zoneout_prob, x, h0, kernel, recurrent_kernel, bias, recurrent_bias,
               zoneout_mask, gamma=None):
    """GRU (gamma None) or LayerNormGRU, reset gate applied after the recurrent product."""
    wx = (x @ kernel if gamma is None else _norm(x @ kernel, gamma[0])) + bias

    def step(t, state):
        (h,) = state
        rh = (h @ recurrent_kernel if gamma is None else _norm(h @ recurrent_kernel, gamma[1])) + recurrent_bias
        xz, xr, xg = torch.chunk(wx[t], 3, dim=1)
        hz, hr, hg = torch.chunk(rh, 3, dim=1)
        z = torch.sigmoid(xz + hz)
        r = torch.sigmoid(xr + hr)
        return (z * h + (1 - z) * torch.tanh(xg + r * hg),)

    return _eager_recurrence(step, (h0,), x.shape[0], training, zoneout_prob, zoneout_mask)[0]


def _eager_indrnn(training, zoneout_prob, x, h0, kernel, recurrent_scale, bias, zoneout_mask, gamma=None):
    """IndRNN (gamma None) or LayerNormIndRNN."""
    wx = (x @ kernel if gamma is None else _norm(x @ kernel, gamma[0])) + bias

    def step(t, state):
        return (torch.tanh(wx[t] + state[0] * recurrent_scale),)

    return _eager_recurrence(step, (h0,), x.shape[0], training, zoneout_prob, zoneout_mask)[0]


def _dropped(weight, mask, scale):
    """The recurrent matrix under DropConnect (what F.dropout gives the reference's loop,
    frameworks/pytorch/lstm.py:263), differentiable with respect to `weight`."""
    return weight if mask is None else weight * mask * scale


# ---- shared layer behaviour (reference frameworks/pytorch/base_rnn.py:25-100) ------------
class _RNNBase(nn.Module):
    _name = "RNN"

    def __init__(self, input_size, hidden_size, batch_first, zoneout, return_state_sequence,
                 dropout=0.0):
        super().__init__()
        if not 0.0 <= dropout <= 1.0:
            raise ValueError("%s: dropout must be in [0.0, 1.0]" % self._name)
        if not 0.0 <= zoneout <= 1.0:
            raise ValueError("%s: zoneout must be in [0.0, 1.0]" % self._name)
        self.input_size = input_size
        self.hidden_size = hidden_size
        self.batch_first = batch_first
        self.zoneout = zoneout
        self.dropout = dropout
        self.return_state_sequence = return_state_sequence

    def _time_major(self, x):
        return x.permute(1, 0, 2) if self.batch_first else x

    def _initial_state(self, x, state, count, fused=False):
        """`count` tensors of shape [N,H]: zeros (None where the fused ops run: they preset them), or
        the caller's [1,N,H] states checked."""
        shape = [1, x.shape[1], self.hidden_size]
        if state is None:
            return (None,) * count if fused else tuple(x.new_zeros(shape[1:]) for _ in range(count))
        states = (state,) if count == 1 else state
        if count > 1 and (not isinstance(states, (tuple, list)) or len(states) != count):
            raise ValueError("RNN state must be a tuple of %d tensors" % count)
        for s in states:
            if not torch.is_tensor(s) or list(s.shape) != shape:
                raise ValueError("RNN state has invalid shape; expected %s, got %s"
                                 % (shape, list(s.shape) if torch.is_tensor(s) else type(s)))
        return tuple(s[0].contiguous() for s in states)

    def _wanted(self, lengths, x):
        """Which states the fused functions are to return (see _wanted_states).  Lengths beyond x are an
        error where the host knows them; on the GPU they give NaNs, for the states and the gradients of their rows."""
        if self.return_state_sequence:
            return "all"
        if lengths is None:
            return "last" if torch.is_grad_enabled() else "last of y"
        lengths = torch.as_tensor(lengths, dtype=torch.long)
        steps = x.shape[0]
        if not lengths.is_cuda and lengths.numel():
            for length in lengths.aminmax():
                if not -steps - 1 <= length <= steps:
                    raise IndexError("length %d is out of bounds for sequences of %d steps" % (length, steps))
        return lengths.to(x.device)

    def _fused_state(self, states, y=None):
        """A state as the layer returns it, from what the fused functions return of it (None: y holds it)."""
        if states is None:
            states = y if self.return_state_sequence else y[-1]
        return (self._time_major(states) if self.return_state_sequence else states).unsqueeze(0)

    def _final_state(self, seq, lengths):
        """seq: [T+1,N,H] state after every step (slot 0 = initial state)."""
        if self.return_state_sequence:
            return self._time_major(seq[1:]).unsqueeze(0)
        if lengths is not None:
            cols = torch.arange(seq.size(1), device=seq.device)
            rows = torch.as_tensor(lengths, device=seq.device, dtype=torch.long)
            return seq[rows, cols].unsqueeze(0)
        return seq[-1].unsqueeze(0)

    def _zoneout_mask(self, x):
        # 1 = take the new value (reference frameworks/pytorch/base_rnn.py:64-70)
        if self.zoneout:
            return x.new_empty(x.shape[0], x.shape[1], self.hidden_size).bernoulli_(1.0 - self.zoneout)
        return None

    def _dropconnect_mask(self, weight):
        """(mask, scale) for inverted dropout on the recurrent matrix, or (None, 1.0)."""
        if not self.training or not self.dropout:
            return None, 1.0
        if self.dropout >= 1.0:
            return torch.zeros_like(weight), 0.0
        keep = 1.0 - self.dropout
        return torch.empty_like(weight).bernoulli_(keep), 1.0 / keep

    def _is_cuda(self):
        """True: the fused GPU ops run; False: the plain torch loop (reference
        frameworks/pytorch/base_rnn.py:72-76)."""
        on_gpu = [t.is_cuda for t in self.parameters()]
        if any(on_gpu) and not all(on_gpu):
            raise ValueError("RNN tensors should all be CUDA tensors or none should be CUDA tensors")
        return any(on_gpu)

    def _check_fused(self, x):
        """What the fused ops need beyond the reference's checks: the input on the GPU and one
        of the dtypes the library is built for, shared by the input and every parameter."""
        tensors = list(self.parameters()) + [x]
        if not x.is_cuda:
            raise RuntimeError("%s: the parameters are GPU tensors, the input must be one too" % self._name)
        if x.dtype not in (torch.float32, torch.float64, torch.float16) or any(t.dtype != x.dtype for t in tensors):
            raise RuntimeError(
                "%s: parameters and input must all have one dtype: float32, float64 or (GRU) float16" % self._name)


def _init_gates(kernel, recurrent_kernel, hidden_size, gates):
    for g in range(gates):
        nn.init.xavier_uniform_(kernel[:, g * hidden_size:(g + 1) * hidden_size])
        nn.init.orthogonal_(recurrent_kernel[:, g * hidden_size:(g + 1) * hidden_size])


def _regroup(w, order_in, order_out):
    """Reorders the gate blocks along the last dimension, e.g. 'igfo' -> 'ifgo'."""
    blocks = dict(zip(order_in, torch.chunk(w, len(order_in), dim=-1)))
    return torch.cat([blocks[g] for g in order_out], dim=-1)


class LSTM(_RNNBase):
    """Long short-term memory layer; gate order i,g,f,o (reference frameworks/pytorch/lstm.py:91-265).

    Parameters: kernel [input_size, 4H] (Xavier uniform per gate), recurrent_kernel [H, 4H]
    (orthogonal per gate), bias [4H] (zeros, forget block = forget_bias).
    """
    _name = "LSTM"

    def __init__(self, input_size, hidden_size, batch_first=False, forget_bias=1.0, dropout=0.0,
                 zoneout=0.0, return_state_sequence=False):
        super().__init__(input_size, hidden_size, batch_first, zoneout, return_state_sequence, dropout)
        self.forget_bias = forget_bias
        self.kernel = nn.Parameter(torch.empty(input_size, hidden_size * 4))
        self.recurrent_kernel = nn.Parameter(torch.empty(hidden_size, hidden_size * 4))
        self.bias = nn.Parameter(torch.empty(hidden_size * 4))
        self.reset_parameters()

    def reset_parameters(self):
        H = self.hidden_size
        with torch.no_grad():
            _init_gates(self.kernel, self.recurrent_kernel, H, 4)
            self.bias.zero_()
            self.bias[2 * H:3 * H].fill_(self.forget_bias)

    def to_native_weights(self):
        """(weight_ih_l0, weight_hh_l0, bias_ih_l0, bias_hh_l0) of an equivalent torch.nn.LSTM."""
        half = _regroup(self.bias.detach(), "igfo", "ifgo") / 2.0
        return (nn.Parameter(_t(_regroup(self.kernel.detach(), "igfo", "ifgo"))),
                nn.Parameter(_t(_regroup(self.recurrent_kernel.detach(), "igfo", "ifgo"))),
                nn.Parameter(half), nn.Parameter(half.clone()))

    def from_native_weights(self, weight_ih_l0, weight_hh_l0, bias_ih_l0, bias_hh_l0):
        """Loads the weights of a torch.nn.LSTM layer."""
        self.kernel = nn.Parameter(_regroup(weight_ih_l0.detach().t(), "ifgo", "igfo").contiguous())
        self.recurrent_kernel = nn.Parameter(_regroup(weight_hh_l0.detach().t(), "ifgo", "igfo").contiguous())
        self.bias = nn.Parameter(_regroup((bias_ih_l0 + bias_hh_l0).detach(), "ifgo", "igfo").contiguous())

    def forward(self, input, state=None, lengths=None):
        """input [T,N,C] ([N,T,C] if batch_first) -> (output, (h_n, c_n)); h_n, c_n are [1,N,H],
        taken at `lengths` when given (the output itself is not masked)."""
        x = self._time_major(input)
        fused = self._is_cuda()
        h0, c0 = self._initial_state(x, state, 2, fused)
        dmask, dscale = self._dropconnect_mask(self.recurrent_kernel)
        zmask = self._zoneout_mask(x)
        if fused:
            self._check_fused(x)
            wanted = self._wanted(lengths, x)
            y, h, c = _LSTMFunction.apply(self.training, self.zoneout, wanted, x.contiguous(), h0, c0,
                                          self.kernel.contiguous(), self.recurrent_kernel.contiguous(),
                                          self.bias.contiguous(), zmask, dmask, dscale)
            return self._time_major(y), (self._fused_state(h, y), self._fused_state(c))
        h, c = _eager_lstm(self.training, self.zoneout, x, h0, c0, self.kernel,
                           _dropped(self.recurrent_kernel, dmask, dscale), self.bias, zmask)
        return self._time_major(h[1:]), (self._final_state(h, lengths), self._final_state(c, lengths))


class GRU(_RNNBase):
    """Gated recurrent unit layer, "reset-after" form, gate order z,r,g (reference
    frameworks/pytorch/gru.py:91-272).  Parameters: kernel [C,3H], recurrent_kernel [H,3H],
    bias [3H], recurrent_bias [3H]."""
    _name = "GRU"

    def __init__(self, input_size, hidden_size, batch_first=False, dropout=0.0, zoneout=0.0,
                 return_state_sequence=False):
        super().__init__(input_size, hidden_size, batch_first, zoneout, return_state_sequence, dropout)
        self.kernel = nn.Parameter(torch.empty(input_size, hidden_size * 3))
        self.recurrent_kernel = nn.Parameter(torch.empty(hidden_size, hidden_size * 3))
        self.bias = nn.Parameter(torch.empty(hidden_size * 3))
        self.recurrent_bias = nn.Parameter(torch.empty(hidden_size * 3))
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            _init_gates(self.kernel, self.recurrent_kernel, self.hidden_size, 3)
            self.bias.zero_()
            self.recurrent_bias.zero_()

    def to_native_weights(self):
        """(weight_ih_l0, weight_hh_l0, bias_ih_l0, bias_hh_l0) of an equivalent torch.nn.GRU."""
        return (nn.Parameter(_t(_regroup(self.kernel.detach(), "zrg", "rzg"))),
                nn.Parameter(_t(_regroup(self.recurrent_kernel.detach(), "zrg", "rzg"))),
                nn.Parameter(_regroup(self.bias.detach(), "zrg", "rzg").contiguous()),
                nn.Parameter(_regroup(self.recurrent_bias.detach(), "zrg", "rzg").contiguous()))

    def from_native_weights(self, weight_ih_l0, weight_hh_l0, bias_ih_l0, bias_hh_l0):
        self.kernel = nn.Parameter(_regroup(weight_ih_l0.detach().t(), "rzg", "zrg").contiguous())
        self.recurrent_kernel = nn.Parameter(_regroup(weight_hh_l0.detach().t(), "rzg", "zrg").contiguous())
        self.bias = nn.Parameter(_regroup(bias_ih_l0.detach(), "rzg", "zrg").contiguous())
        self.recurrent_bias = nn.Parameter(_regroup(bias_hh_l0.detach(), "rzg", "zrg").contiguous())

    def forward(self, input, state=None, lengths=None):
        x = self._time_major(input)
        fused = self._is_cuda()
        (h0,) = self._initial_state(x, state, 1, fused)
        dmask, dscale = self._dropconnect_mask(self.recurrent_kernel)
        zmask = self._zoneout_mask(x)
        if fused:
            self._check_fused(x)
            wanted = self._wanted(lengths, x)
            y, h = _GRUFunction.apply(self.training, self.zoneout, wanted, x.contiguous(), h0,
                                      self.kernel.contiguous(), self.recurrent_kernel.contiguous(),
                                      self.bias.contiguous(), self.recurrent_bias.contiguous(),
                                      zmask, dmask, dscale)
            return self._time_major(y), self._fused_state(h, y)
        h = _eager_gru(self.training, self.zoneout, x, h0, self.kernel,
                       _dropped(self.recurrent_kernel, dmask, dscale), self.bias,
                       self.recurrent_bias, zmask)
        return self._time_major(h[1:]), self._final_state(h, lengths)


class IndRNN(_RNNBase):
    """Independently recurrent layer h' = tanh(xW + u*h + b) (reference
    frameworks/pytorch/indrnn.py:78-190).  Parameters: kernel [C,H], recurrent_scale [H]
    (uniform in [-0.5, 0.5]), bias [H]."""
    _name = "IndRNN"

    def __init__(self, input_size, hidden_size, batch_first=False, zoneout=0.0,
                 return_state_sequence=False):
        super().__init__(input_size, hidden_size, batch_first, zoneout, return_state_sequence)
        self.kernel = nn.Parameter(torch.empty(input_size, hidden_size))
        self.recurrent_scale = nn.Parameter(torch.empty(hidden_size))
        self.bias = nn.Parameter(torch.empty(hidden_size))
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            nn.init.xavier_uniform_(self.kernel)
            nn.init.uniform_(self.recurrent_scale, -0.5, 0.5)
            self.bias.zero_()

    def forward(self, input, state=None, lengths=None):
        x = self._time_major(input)
        fused = self._is_cuda()
        (h0,) = self._initial_state(x, state, 1, fused)
        zmask = self._zoneout_mask(x)
        if fused:
            self._check_fused(x)
            wanted = self._wanted(lengths, x)
            y, h = _IndRNNFunction.apply(self.training, self.zoneout, wanted, x.contiguous(), h0,
                                         self.kernel.contiguous(), self.recurrent_scale.contiguous(),
                                         self.bias.contiguous(), zmask)
            return self._time_major(y), self._fused_state(h, y)
        h = _eager_indrnn(self.training, self.zoneout, x, h0, self.kernel, self.recurrent_scale,
                          self.bias, zmask)
        return self._time_major(h[1:]), self._final_state(h, lengths)


class LayerNormIndRNN(_RNNBase):
    """IndRNN with layer norm on the input projection (reference
    frameworks/pytorch/layer_norm_indrnn.py:83-203); gamma is [2,H], only row 0 is used."""
    _name = "LayerNormIndRNN"

    def __init__(self, input_size, hidden_size, batch_first=False, zoneout=0.0,
                 return_state_sequence=False):
        super().__init__(input_size, hidden_size, batch_first, zoneout, return_state_sequence)
        self.kernel = nn.Parameter(torch.empty(input_size, hidden_size))
        self.recurrent_scale = nn.Parameter(torch.empty(hidden_size))
        self.bias = nn.Parameter(torch.empty(hidden_size))
        self.gamma = nn.Parameter(torch.empty(2, hidden_size))
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            nn.init.xavier_uniform_(self.kernel)
            nn.init.uniform_(self.recurrent_scale, -0.5, 0.5)
            self.bias.zero_()
            self.gamma.fill_(1.0)

    def forward(self, input, state=None, lengths=None):
        x = self._time_major(input)
        fused = self._is_cuda()
        (h0,) = self._initial_state(x, state, 1, fused)
        zmask = self._zoneout_mask(x)
        if fused:
            self._check_fused(x)
            wanted = self._wanted(lengths, x)
            y, h = _LayerNormIndRNNFunction.apply(self.training, self.zoneout, wanted, x.contiguous(), h0,
                                                  self.kernel.contiguous(), self.recurrent_scale.contiguous(),
                                                  self.bias.contiguous(), self.gamma.contiguous(), zmask)
            return self._time_major(y), self._fused_state(h, y)
        h = _eager_indrnn(self.training, self.zoneout, x, h0, self.kernel, self.recurrent_scale,
                          self.bias, zmask, gamma=self.gamma)
        return self._time_major(h[1:]), self._final_state(h, lengths)


class LayerNormLSTM(_RNNBase):
    """LSTM with layer norm on xW, on hR and on the cell state (reference
    frameworks/pytorch/layer_norm_lstm.py:94-245).  Extra parameters: gamma [2,4H] (ones),
    gamma_h [H] (ones), beta_h [H] (zeros)."""
    _name = "LayerNormLSTM"

    def __init__(self, input_size, hidden_size, batch_first=False, forget_bias=1.0, dropout=0.0,
                 zoneout=0.0, return_state_sequence=False):
        super().__init__(input_size, hidden_size, batch_first, zoneout, return_state_sequence, dropout)
        self.forget_bias = forget_bias
        self.kernel = nn.Parameter(torch.empty(input_size, hidden_size * 4))
        self.recurrent_kernel = nn.Parameter(torch.empty(hidden_size, hidden_size * 4))
        self.bias = nn.Parameter(torch.empty(hidden_size * 4))
        self.gamma = nn.Parameter(torch.empty(2, hidden_size * 4))
        self.gamma_h = nn.Parameter(torch.empty(hidden_size))
        self.beta_h = nn.Parameter(torch.empty(hidden_size))
        self.reset_parameters()

    def reset_parameters(self):
        H = self.hidden_size
        with torch.no_grad():
            _init_gates(self.kernel, self.recurrent_kernel, H, 4)
            self.bias.zero_()
            self.bias[2 * H:3 * H].fill_(self.forget_bias)
            self.gamma.fill_(1.0)
            self.gamma_h.fill_(1.0)
            self.beta_h.zero_()

    def forward(self, input, state=None, lengths=None):
        x = self._time_major(input)
        fused = self._is_cuda()
        h0, c0 = self._initial_state(x, state, 2, fused)
        dmask, dscale = self._dropconnect_mask(self.recurrent_kernel)
        R = _dropped(self.recurrent_kernel, dmask, dscale)
        zmask = self._zoneout_mask(x)
        if fused:
            self._check_fused(x)
            wanted = self._wanted(lengths, x)
            y, h, c = _LayerNormLSTMFunction.apply(self.training, self.zoneout, wanted, x.contiguous(), h0, c0,
                                                   self.kernel.contiguous(), R.contiguous(),
                                                   self.bias.contiguous(), self.gamma.contiguous(),
                                                   self.gamma_h.contiguous(), self.beta_h.contiguous(), zmask)
            return self._time_major(y), (self._fused_state(h, y), self._fused_state(c))
        h, c = _eager_lstm(self.training, self.zoneout, x, h0, c0, self.kernel, R, self.bias, zmask,
                           gamma=self.gamma, gamma_h=self.gamma_h, beta_h=self.beta_h)
        return self._time_major(h[1:]), (self._final_state(h, lengths), self._final_state(c, lengths))


class LayerNormGRU(_RNNBase):
    """GRU with layer norm on xW and on hR (reference frameworks/pytorch/layer_norm_gru.py:94-233);
    gamma is [2,3H] (ones)."""
    _name = "LayerNormGRU"

    def __init__(self, input_size, hidden_size, batch_first=False, dropout=0.0, zoneout=0.0,
                 return_state_sequence=False):
        super().__init__(input_size, hidden_size, batch_first, zoneout, return_state_sequence, dropout)
        self.kernel = nn.Parameter(torch.empty(input_size, hidden_size * 3))
        self.recurrent_kernel = nn.Parameter(torch.empty(hidden_size, hidden_size * 3))
        self.bias = nn.Parameter(torch.empty(hidden_size * 3))
        self.recurrent_bias = nn.Parameter(torch.empty(hidden_size * 3))
        self.gamma = nn.Parameter(torch.empty(2, hidden_size * 3))
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            _init_gates(self.kernel, self.recurrent_kernel, self.hidden_size, 3)
            self.bias.zero_()
            self.recurrent_bias.zero_()
            self.gamma.fill_(1.0)

    def forward(self, input, state=None, lengths=None):
        x = self._time_major(input)
        fused = self._is_cuda()
        (h0,) = self._initial_state(x, state, 1, fused)
        dmask, dscale = self._dropconnect_mask(self.recurrent_kernel)
        R = _dropped(self.recurrent_kernel, dmask, dscale)
        zmask = self._zoneout_mask(x)
        if fused:
            self._check_fused(x)
            wanted = self._wanted(lengths, x)
            y, h = _LayerNormGRUFunction.apply(self.training, self.zoneout, wanted, x.contiguous(), h0,
                                               self.kernel.contiguous(), R.contiguous(),
                                               self.bias.contiguous(), self.recurrent_bias.contiguous(),
                                               self.gamma.contiguous(), zmask)
            return self._time_major(y), self._fused_state(h, y)
        h = _eager_gru(self.training, self.zoneout, x, h0, self.kernel, R, self.bias,
                       self.recurrent_bias, zmask, gamma=self.gamma)
        return self._time_major(h[1:]), self._final_state(h, lengths)


# ---- the layers of a state space block ---------------------------------------------------
# Projections between them are the caller's.  Parameters are handed over in float32 whatever they are kept in (their
# gradients come back in the type they have); activations keep theirs.
class _CausalConvFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kernel, bias, silu, state, lengths):
        ctx.save_for_backward(x, kernel, bias, state, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return ops.causal_conv_forward(x, kernel, bias, silu, state, lengths)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dstate_out):
        x, kernel, bias, state, lengths = ctx.saved_tensors
        dx, dkernel, dbias, dstate = ops.causal_conv_backward(x, kernel, bias, ctx.silu, state, lengths, dy, dstate_out)
        return dx, dkernel, dbias, None, dstate, None


class _SelectiveScanFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, training, x, delta, A, B, C, D, z, delta_bias, delta_softplus, h0, lengths):
        y, h_last, cache = ops.selective_scan_forward(training and any(ctx.needs_input_grad), x, delta, A, B, C, D, z, delta_bias,
                                                      delta_softplus, h0, lengths)
        ctx.save_for_backward(x, delta, A, B, C, D, z, delta_bias, lengths, cache)
        ctx.delta_softplus, ctx.has_h0 = delta_softplus, h0 is not None
        ctx.set_materialize_grads(False)
        return y, h_last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh_last):
        x, delta, A, B, C, D, z, delta_bias, lengths, cache = ctx.saved_tensors
        dx, ddelta, dA, dB, dC, dD, dz, dbias, dh0 = ops.selective_scan_backward(
            x, delta, A, B, C, D, z, delta_bias, ctx.delta_softplus, None, lengths, cache, dy, dh_last)
        return None, dx, ddelta, dA, dB, dC, dD, dz, dbias, None, dh0 if ctx.has_h0 else None, None


class _ResidualNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, update, residual, gate, scale, after_weight, before_weight, before_bias, centered, eps):
        out, normed, stats = ops.residual_norm_forward(update, residual, gate, scale, after_weight, before_weight, before_bias,
                                                       centered, eps)
        ctx.save_for_backward(update, residual, gate, scale, after_weight, before_weight, before_bias, stats)
        ctx.centered = centered
        ctx.set_materialize_grads(False)
        return out, normed

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dnormed):
        return (*ops.residual_norm_backward(*ctx.saved_tensors, dout, dnormed, centered=ctx.centered), None, None)


def _wide(*tensors):
    """Half types as float32; what the plain forms compute in."""
    return tuple(t if t is None or t.dtype in (torch.float32, torch.float64) else t.float() for t in tensors)


def _inside(lengths, T, N, like):
    """[T,N]: the steps that belong to the rows' sequences."""
    steps = torch.arange(T, device=like.device)[:, None]
    return steps < (torch.full((N,), T, device=like.device) if lengths is None else torch.where(lengths < 0, lengths + T + 1, lengths))


def _eager_causal_conv(x, kernel, bias, silu, state, lengths):
    dtype, (T, N, D), W = x.dtype, x.shape, kernel.shape[0]
    x, kernel, bias, state = _wide(x, kernel, bias, state)
    inside = _inside(lengths, T, N, x)
    x = torch.where(inside[..., None], x, 0.0)
    padded = torch.cat([x.new_zeros(W - 1, N, D) if state is None else state, x])
    pre = sum(kernel[k] * padded[k:k + T] for k in range(W))
    pre = pre if bias is None else pre + bias
    y = torch.where(inside[..., None], F.silu(pre) if silu else pre, 0.0)
    rows = inside.sum(0) + torch.arange(W - 1, device=x.device)[:, None]
    return y.to(dtype), padded[rows, torch.arange(N, device=x.device)].to(dtype)


def _eager_selective_scan(x, delta, A, B, C, D, z, delta_bias, delta_softplus, h0, lengths):
    dtype, (T, N, channels) = x.dtype, x.shape
    x, delta, A, B, C, D, z, delta_bias, h = _wide(x, delta, A, B, C, D, z, delta_bias, h0)
    inside = _inside(lengths, T, N, x)
    x, delta, z = (t if t is None else torch.where(inside[..., None], t, 0.0) for t in (x, delta, z))
    B, C = (torch.where(inside[..., None, None], t if t.dim() == 4 else t.unsqueeze(2), 0.0) for t in (B, C))
    share = channels // B.shape[2]
    dt = delta if delta_bias is None else delta + delta_bias
    dt = F.softplus(dt, threshold=50.0) if delta_softplus else dt
    h = x.new_zeros(N, channels, A.shape[1]) if h is None else h
    ys = []
    for t in range(T):
        new = torch.exp(dt[t, :, :, None] * A) * h + (dt[t] * x[t])[..., None] * B[t].repeat_interleave(share, 1)
        y = (new * C[t].repeat_interleave(share, 1)).sum(-1)
        h = torch.where(inside[t][:, None, None], new, h)
        ys.append(y if D is None else y + D * x[t])
    y = torch.stack(ys)
    y = y if z is None else y * F.silu(z)
    return torch.where(inside[..., None], y, 0.0).to(dtype), h


def _eager_residual_norm(update, residual, gate, scale, after_weight, before_weight, before_bias, centered, eps):
    dtype = update.dtype
    v, residual, gate, scale, after, before, bias = _wide(update, residual, gate, scale, after_weight, before_weight, before_bias)

    def norm(v):
        v = v - v.mean(-1, keepdim=True) if centered else v
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps)

    v = v if after is None else norm(v) * after
    v = v if gate is None else v * F.silu(gate)
    v = v if scale is None else v * scale
    v = v if residual is None else v + residual
    n = None if before is None else norm(v) * before
    n = n if bias is None else n + bias
    return v.to(dtype), None if n is None else n.to(dtype)


class _BlockLayer(nn.Module):
    """What the layers of a state space block share."""
    _name = "layer"

    def _fused(self, x):
        """Whether the fused ops run, decided and checked as the recurrent layers do."""
        fused = _RNNBase._is_cuda(self)
        if fused and not x.is_cuda:
            raise RuntimeError("%s: the parameters are GPU tensors, the input must be one too" % self._name)
        if fused and x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise RuntimeError("%s: the input must be float32, float16 or bfloat16" % self._name)
        return fused

    def _rows(self, t):
        return t.transpose(0, 1) if t is not None and getattr(self, "batch_first", False) else t

    def _lengths(self, lengths, x):
        """int64 [N] on the input's device.  Lengths beyond x are an error where the host knows them; on the GPU they give NaNs."""
        if lengths is None:
            return None
        lengths = torch.as_tensor(lengths, dtype=torch.long)
        steps = x.shape[0]
        if not lengths.is_cuda and lengths.numel():
            for length in lengths.aminmax():
                if not -steps - 1 <= length <= steps:
                    raise IndexError("length %d is out of bounds for sequences of %d steps" % (length, steps))
        if tuple(lengths.shape) != (x.shape[1],):
            raise ValueError("%s: lengths must be [%d], got %s" % (self._name, x.shape[1], list(lengths.shape)))
        return lengths.to(x.device).contiguous()


def _as_float(p):
    return p if p is None or p.dtype == torch.float32 else p.float()


class CausalConv(_BlockLayer):
    """Short causal convolution over time, one filter per channel: y[t] = act(bias + sum_k kernel[k] x[t-width+1+k]),
    act(v) = v sigmoid(v) with silu.  Parameters: kernel [width, channels], bias [channels] (uniform in
    +-width^-0.5).  width of 1 to 8."""
    _name = "CausalConv"

    def __init__(self, channels, width=4, bias=True, silu=True, batch_first=False):
        super().__init__()
        if not 1 <= width <= 8:
            raise ValueError("%s: width must be in [1, 8]" % self._name)
        self.channels, self.width, self.silu, self.batch_first = channels, width, silu, batch_first
        self.kernel = nn.Parameter(torch.empty(width, channels))
        self.bias = nn.Parameter(torch.empty(channels)) if bias else None
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            for p in self.parameters():
                p.uniform_(-self.width ** -0.5, self.width ** -0.5)

    def forward(self, input, state=None, lengths=None):
        """input [T,N,channels] ([N,T,channels] if batch_first) -> (output, state): state [width-1,N,channels] holds the
        inputs before the first step (None: zeros), and is returned for the step behind the last (of the row's
        length).  Outputs behind a row's length are 0."""
        x = self._rows(input)
        lengths = self._lengths(lengths, x)
        if self._fused(x):
            y, state = _CausalConvFunction.apply(x, _as_float(self.kernel), _as_float(self.bias), self.silu, state, lengths)
        else:
            y, state = _eager_causal_conv(x, self.kernel, self.bias, self.silu, state, lengths)
        return self._rows(y), state

    def step(self, input, state=None):
        """One step without gradients: input [N,channels] -> (output, state)."""
        with torch.no_grad():
            if state is None:
                state = input.new_zeros((self.width - 1, *input.shape))
            if self._fused(input):
                return ops.causal_conv_iterate(input, state, _as_float(self.kernel), _as_float(self.bias), self.silu)
            y, state = _eager_causal_conv(input.unsqueeze(0), self.kernel, self.bias, self.silu, state, None)
            return y[0], state


class SelectiveScan(_BlockLayer):
    """Selective state space recurrence: with A = -exp(log_decay) and dt = softplus(delta + delta_bias),
    h[t] = exp(dt A) h[t-1] + dt x B, y = (sum_s C h + skip x) silu(z).  Parameters: log_decay [channels, state_size]
    (logarithms of 1 .. state_size), skip [channels] (ones), delta_bias [channels] (step sizes of 0.001 to 0.1).  `groups`
    groups of channels share B and C; state_size of 1 to 64."""
    _name = "SelectiveScan"

    def __init__(self, channels, state_size=16, groups=1, batch_first=False):
        super().__init__()
        if not 1 <= state_size <= 64:
            raise ValueError("%s: state_size must be in [1, 64]" % self._name)
        if groups < 1 or channels % groups:
            raise ValueError("%s: %d channels cannot be shared by %d groups" % (self._name, channels, groups))
        self.channels, self.state_size, self.groups, self.batch_first = channels, state_size, groups, batch_first
        self.log_decay = nn.Parameter(torch.empty(channels, state_size))
        self.skip = nn.Parameter(torch.empty(channels))
        self.delta_bias = nn.Parameter(torch.empty(channels))
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            self.log_decay.copy_(torch.log(torch.arange(1.0, self.state_size + 1)).expand_as(self.log_decay))
            self.skip.fill_(1.0)
            dt = torch.exp(torch.empty_like(self.delta_bias, dtype=torch.float32).uniform_(-6.907755, -2.302585))
            self.delta_bias.copy_(dt + torch.log(-torch.expm1(-dt)))

    def _decay(self):
        return -torch.exp(_as_float(self.log_decay) if self.log_decay.dtype != torch.float64 else self.log_decay)

    def _grouped(self, t):
        return t.unflatten(-1, (self.groups, self.state_size))

    def forward(self, x, delta, B, C, z=None, state=None, lengths=None):
        """x, delta, z [T,N,channels], B, C [T,N,groups*state_size] ([N,T,*] if batch_first) -> (output, state): state
        [N,channels,state_size], float32, before the first step (None: zeros) and after the last (of the row's length).
        Outputs behind a row's length are 0."""
        x, delta, B, C, z = (self._rows(t) for t in (x, delta, B, C, z))
        lengths = self._lengths(lengths, x)
        arguments = x, delta, self._decay(), self._grouped(B), self._grouped(C)
        if self._fused(x):
            y, state = _SelectiveScanFunction.apply(torch.is_grad_enabled(), *arguments, _as_float(self.skip), z,
                                                    _as_float(self.delta_bias), True, state, lengths)
        else:
            y, state = _eager_selective_scan(*arguments, self.skip, z, self.delta_bias, True, state, lengths)
        return self._rows(y), state

    def step(self, x, delta, B, C, z=None, state=None):
        """One step without gradients: x, delta, z [N,channels], B, C [N,groups*state_size] -> (output, state)."""
        with torch.no_grad():
            if state is None:
                state = torch.zeros(x.shape[0], self.channels, self.state_size, device=x.device,
                                    dtype=x.dtype if x.dtype == torch.float64 else torch.float32)
            arguments = x, delta, self._decay(), self._grouped(B), self._grouped(C)
            if self._fused(x):
                return ops.selective_scan_iterate(*arguments, state, _as_float(self.skip), z, _as_float(self.delta_bias), True)
            x, delta, A, B, C = (t if t is arguments[2] else t.unsqueeze(0) for t in arguments)
            y, state = _eager_selective_scan(x, delta, A, B, C, self.skip, None if z is None else z.unsqueeze(0),
                                             self.delta_bias, True, state, None)
            return y[0], state


class ResidualNorm(_BlockLayer):
    """The norms around a block, its gate and its residual scale: out = residual + scale norm(update) after_weight silu(gate),
    normed = norm(out) before_weight + before_bias, of which `out` leaves the block and `normed` enters the next one.  norm is
    the root mean square norm, or layer norm (centered).  Parameters, each [channels]: after_weight (ones; absent unless
    norm_after), scale (`scale`; absent if None), before_weight (ones; absent unless norm_before), before_bias (zeros; centered
    only).  At most 8192 channels."""
    _name = "ResidualNorm"

    def __init__(self, channels, centered=False, norm_after=True, norm_before=True, scale=1.0, eps=1e-5):
        super().__init__()
        self.channels, self.centered, self.eps, self.initial_scale = channels, centered, eps, scale
        make = lambda wanted: nn.Parameter(torch.empty(channels)) if wanted else None  # noqa: E731
        self.after_weight = make(norm_after)
        self.scale = make(scale is not None)
        self.before_weight = make(norm_before)
        self.before_bias = make(norm_before and centered)
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            for p, value in ((self.after_weight, 1.0), (self.scale, self.initial_scale), (self.before_weight, 1.0),
                             (self.before_bias, 0.0)):
                if p is not None:
                    p.fill_(value)

    def forward(self, update, residual=None, gate=None):
        """Tensors [T,N,channels] (in whatever order, or [N,channels]) -> (out, normed); normed is None unless norm_before."""
        weights = self.scale, self.after_weight, self.before_weight, self.before_bias
        if self._fused(update) or update.is_cuda and not list(self.parameters()):
            return _ResidualNormFunction.apply(update, residual, gate, *map(_as_float, weights), self.centered, self.eps)
        return _eager_residual_norm(update, residual, gate, *weights, self.centered, self.eps)


# ---- the layers of a gated linear recurrent block, and the clipping of gradients ----------------------
class _LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, training, x, kernel, bias, activation, residual):
        y, cache = ops.linear_forward(training and any(ctx.needs_input_grad), x, kernel, bias, activation, residual)
        ctx.save_for_backward(x, kernel, bias, cache)
        ctx.activation, ctx.has_residual = activation, residual is not None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, kernel, bias, cache = ctx.saved_tensors
        wanted = ctx.needs_input_grad
        dx = dkernel = dbias = None
        if any(wanted[1:4]):
            dx, dkernel, dbias = ops.linear_backward(x, kernel, bias, ctx.activation, cache, dy, wanted[1], wanted[2])
        return None, dx, dkernel, dbias, None, dy if ctx.has_residual else None


class _GatedRecurrenceFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, training, x, forget, admit, z, decay, forget_bias, admit_bias, h0, lengths):
        y, h_last, cache = ops.gated_recurrence_forward(training and any(ctx.needs_input_grad), x, forget, admit, z, decay, forget_bias,
                                                        admit_bias, h0, lengths)
        ctx.save_for_backward(x, forget, admit, z, decay, forget_bias, admit_bias, h0, lengths, cache)
        ctx.set_materialize_grads(False)
        return y, h_last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh_last):
        return (None, *ops.gated_recurrence_backward(*ctx.saved_tensors, dy, dh_last), None)


def _eager_linear(x, kernel, bias, activation, residual):
    dtype = x.dtype
    x, kernel, bias, residual = _wide(x, kernel, bias, residual)
    y = x @ kernel if bias is None else x @ kernel + bias
    y = {"none": lambda v: v, "gelu": F.gelu, "silu": F.silu}[activation](y)
    return (y if residual is None else y + residual).to(dtype)


def _eager_gated_recurrence(x, forget, admit, z, decay, forget_bias, admit_bias, h0, lengths):
    dtype, (T, N, D) = x.dtype, x.shape
    x, forget, admit, z, decay, forget_bias, admit_bias, h = _wide(x, forget, admit, z, decay, forget_bias, admit_bias, h0)
    inside = _inside(lengths, T, N, x)[..., None]
    x, forget, admit, z = (t if t is None else torch.where(inside, t, 0.0) for t in (x, forget, admit, z))
    raw = forget if forget_bias is None else forget + forget_bias
    r = torch.sigmoid(raw)
    i = None if admit is None else torch.sigmoid(admit if admit_bias is None else admit + admit_bias)
    fed = x if i is None else x * i
    if decay is None:
        a, u = r, fed if i is not None else torch.sigmoid(-raw) * x
    else:
        a, u = torch.exp(-decay * r), torch.sqrt(-torch.expm1(-2 * decay * r)) * fed
    h = x.new_zeros(N, D) if h is None else h
    ys = []
    for t in range(T):
        h = torch.where(inside[t], a[t] * h + u[t], h)
        ys.append(h)
    y = torch.stack(ys)
    y = y if z is None else y * F.silu(z)
    return torch.where(inside, y, 0.0).to(dtype), h


class Linear(_BlockLayer):
    """A projection with what follows it: act(input kernel + bias) + residual.  activation: "none", "gelu" (v times the normal
    distribution function) or "silu" (v sigmoid(v)).  Parameters: kernel [inputs, outputs] (uniform in +-sqrt(6 / (inputs + outputs))),
    bias [outputs] (zeros); they are handed over in the input's type, and their gradients come back in the type they have."""
    _name = "Linear"

    def __init__(self, inputs, outputs, bias=True, activation="none"):
        super().__init__()
        if activation not in ("none", "gelu", "silu"):
            raise ValueError("%s: activation must be none, gelu or silu, got %r" % (self._name, activation))
        self.inputs, self.outputs, self.activation = inputs, outputs, activation
        self.kernel = nn.Parameter(torch.empty(inputs, outputs))
        self.bias = nn.Parameter(torch.empty(outputs)) if bias else None
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            nn.init.xavier_uniform_(self.kernel)
            if self.bias is not None:
                self.bias.zero_()

    def forward(self, input, residual=None):
        """input [T,N,inputs] (in whatever order, or [N,inputs]), residual [T,N,outputs] -> [T,N,outputs]."""
        kernel, bias = self.kernel, self.bias
        if self._fused(input):
            return _LinearFunction.apply(torch.is_grad_enabled(), input, kernel.to(input.dtype),
                                         None if bias is None else bias.to(input.dtype), self.activation, residual)
        return _eager_linear(input, kernel, bias, self.activation, residual)


class GatedRecurrence(_BlockLayer):
    """Gated linear recurrence, one state a channel: with r = sigmoid(forget + forget_bias), i = sigmoid(admit + admit_bias)
    h[t] = a h[t-1] + sqrt(1 - a^2) i x with a = exp(-exp(log_decay) r), or (decay=False) h[t] = r h[t-1] + i x;  output h silu(z).
    admit=False: no gate on inputs, i = 1 (without a decay i = 1 - r).  Parameters, each [channels]: log_decay (decays of
    0.81 to 0.998 under an open gate), forget_bias (zeros; without a decay from 0.5 to 6), admit_bias (zeros)."""
    _name = "GatedRecurrence"

    def __init__(self, channels, decay=True, admit=True, batch_first=False):
        super().__init__()
        self.channels, self.batch_first = channels, batch_first
        self.log_decay = nn.Parameter(torch.empty(channels)) if decay else None
        self.forget_bias = nn.Parameter(torch.empty(channels))
        self.admit_bias = nn.Parameter(torch.empty(channels)) if admit else None
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            if self.log_decay is not None:
                self.log_decay.copy_(torch.log(-2 * torch.log(torch.empty_like(self.log_decay, dtype=torch.float32).uniform_(0.9, 0.999))))
                self.forget_bias.zero_()
            else:
                self.forget_bias.uniform_(0.5, 6.0)
            if self.admit_bias is not None:
                self.admit_bias.zero_()

    def _arguments(self, x, forget, admit, z):
        if (admit is None) != (self.admit_bias is None):
            raise ValueError("%s: admit must be %s" % (self._name, "left out" if self.admit_bias is None else "given"))
        fused = self._fused(x)
        of = _as_float if fused else lambda p: p
        decay = None if self.log_decay is None else torch.exp(of(self.log_decay))
        return fused, (x, forget, admit, z, decay, of(self.forget_bias), of(self.admit_bias))

    def forward(self, x, forget, admit=None, z=None, state=None, lengths=None):
        """x, forget, admit, z [T,N,channels] ([N,T,channels] if batch_first) -> (output, state): state [N,channels], float32,
        before the first step (None: zeros) and after the last (of the row's length).  Outputs behind a row's length are 0."""
        x, forget, admit, z = (self._rows(t) for t in (x, forget, admit, z))
        lengths = self._lengths(lengths, x)
        fused, arguments = self._arguments(x, forget, admit, z)
        if fused:
            y, state = _GatedRecurrenceFunction.apply(torch.is_grad_enabled(), *arguments, state, lengths)
        else:
            y, state = _eager_gated_recurrence(*arguments, state, lengths)
        return self._rows(y), state

    def step(self, x, forget, admit=None, z=None, state=None):
        """One step without gradients: x, forget, admit, z [N,channels] -> (output, state)."""
        with torch.no_grad():
            if state is None:
                state = torch.zeros(x.shape, device=x.device, dtype=x.dtype if x.dtype == torch.float64 else torch.float32)
            fused, arguments = self._arguments(x, forget, admit, z)
            if fused:
                return ops.gated_recurrence_iterate(*arguments[:2], state, *arguments[2:])
            steps = (t if t is None else t.unsqueeze(0) for t in arguments[:4])
            y, state = _eager_gated_recurrence(*steps, *arguments[4:], state, None)
            return y[0], state


def clip_gradients_(parameters, max_norm):
    """Scales the gradients of `parameters` (a tensor or several; those without one are left out, and one that is listed more than
    once, as tied weights may be, counts once) in place so that their norm together is at most max_norm: each times
    min(1, max_norm / (norm + 1e-6)).  Returns the norm before, a tensor of no axes; on the GPU nothing is waited for.  Gradients of
    float32, float64, float16 and bfloat16 may be mixed; they are on one device, and on the GPU each fills its memory, as those that
    autograd makes do, and shares it with no other."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    grads = list({id(g): g for g in grads}.values())
    if not grads:
        return torch.zeros(())
    with torch.no_grad():
        if grads[0].is_cuda:
            return ops.clip_gradients(grads, max_norm, out=grads)[1]
        if any(g.is_cuda for g in grads):
            raise ValueError("gradients must be on one device")
        if not float(max_norm) >= 0:
            raise ValueError("max_norm must not be below 0, got %r" % max_norm)
        wide = torch.float64 if any(g.dtype == torch.float64 for g in grads) else torch.float32
        whole = torch.sqrt(sum(g.double().square().sum() for g in grads))
        norm = whole.to(wide)
        factor = (float(max_norm) / ((norm.double() if norm.isfinite() else whole) + 1e-6)).clamp(max=1.0)
        for g in grads:  # (a factor below a float's normal range would lose bits, or all, as one)
            g.copy_(g.double() * factor if g.dtype == torch.float64 or factor < 2.0 ** -126 else g.float() * factor.float())
        return norm
