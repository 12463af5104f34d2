"""Python mirror of the C kernel API (include/pulpnn_b200.h), one function per reference entry
point with the reference's argument order (32bit/include/pulp_nn_kernels.h) preceded by the
batch-norm width ``bits`` (32 or 64) that selects the tree.

Buffers may be torch tensors (CUDA or CPU), numpy arrays or raw integer addresses; what reaches
the library is the address. Device memory is used in place; host memory is staged by the
library itself. Errors recorded by the library are raised as ``PulpNNError``.
"""
import ctypes as C
import struct

import numpy as np

from . import _lib

OK, ERR_INVALID_ARG, ERR_UNSUPPORTED, ERR_CUDA, ERR_NO_DEVICE, ERR_DEVICE_WAIT = range(6)
OPT_FORCE_GENERIC, OPT_MAXPOOL_CLOBBER, OPT_SPLIT_K, OPT_FUSE_DWPW, OPT_TUNE = 1, 2, 3, 4, 5
LAYER_CONV, LAYER_POINTWISE, LAYER_DEPTHWISE, LAYER_AVGPOOL, LAYER_MAXPOOL, LAYER_LINEAR_OUT_32 = range(6)


class PulpNNError(RuntimeError):
    def __init__(self, code, message):
        super().__init__("pulpnn error %d: %s" % (code, message))
        self.code = code


def _ptr(x):
    """Address of a buffer (torch tensor, numpy array, int or None)."""
    if x is None:
        return None
    if isinstance(x, int):
        return C.c_void_p(x)
    if isinstance(x, np.ndarray):
        assert x.flags["C_CONTIGUOUS"], "buffers must be contiguous"
        return C.c_void_p(x.ctypes.data)
    if hasattr(x, "data_ptr"):
        assert x.is_contiguous(), "buffers must be contiguous"
        return C.c_void_p(x.data_ptr())
    raise TypeError("unsupported buffer type %r" % type(x))


def _check():
    lib = _lib.load_library()
    code = lib.pulpnn_last_error()
    if code != OK:
        msg = lib.pulpnn_last_error_message().decode()
        lib.pulpnn_clear_error()
        raise PulpNNError(code, msg)


def _sfx(bits):
    if bits not in (32, 64):
        raise ValueError("bits must be 32 or 64")
    return "_bn%d" % bits


def _fn(name, bits):
    f = getattr(_lib.load_library(), name + _sfx(bits))
    f.restype = None
    return f


# ---- context ------------------------------------------------------------------------------
def set_device(index):
    if _lib.load_library().pulpnn_set_device(int(index)) != OK:
        _check()


def set_stream(stream):
    """stream: None (default stream), an integer cudaStream_t or a torch.cuda.Stream."""
    handle = 0 if stream is None else int(getattr(stream, "cuda_stream", stream))
    _lib.load_library().pulpnn_set_stream(C.c_void_p(handle))


def set_batch(n):
    if _lib.load_library().pulpnn_set_batch(int(n)) != OK:
        _check()


def get_batch():
    return _lib.load_library().pulpnn_get_batch()


def synchronize():
    if _lib.load_library().pulpnn_synchronize() != OK:
        _check()


def launch_count():
    return int(_lib.load_library().pulpnn_launch_count())


def last_kernel():
    """Kernel family of this thread's latest launch."""
    return _lib.load_library().pulpnn_last_kernel().decode()


def device_status():
    return _lib.load_library().pulpnn_device_status()


def set_option(option, value):
    if _lib.load_library().pulpnn_set_option(int(option), int(value)) != OK:
        _check()


def get_option(option):
    return _lib.load_library().pulpnn_get_option(int(option))


# ---- calls with packed arguments (csrc/packed_calls.cu) ----------------------------------------
# The common case of every entry point: arguments that struct packs as they are go over as one block of bytes.
# Whatever it does not take (a value that the C type cuts, an object without an integer) goes argument by argument,
# with the conversions and errors of ctypes.
def _addr(x):
    """Address of a buffer as an integer, 0 for None."""
    if x is None:
        return 0
    try:
        a = x.data_ptr()
    except AttributeError:
        return _ptr(x).value or 0
    assert x.is_contiguous(), "buffers must be contiguous"
    return a


class _Packed:
    """call(bits, ...) of one packed entry point; `through` names the entry it forwards to, if it serves several."""

    def __init__(self, name, fmt, through=None):
        self.name, self.pack, self.through, self.bound = name, struct.Struct(fmt).pack, through, {}

    def bind(self, bits):
        f = getattr(_lib.load_library(), "pulpnn_packed_" + self.name + _sfx(bits))
        f.restype = C.c_int
        if self.through is None:
            f.argtypes = [C.c_char_p]
            call = f
        else:
            # the library's functions are shared objects of ctypes: a prototype of our own leaves theirs alone
            proto = C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_char_p)
            fn = proto(C.cast(f, C.c_void_p).value)
            entry = C.cast(_fn(self.through, bits), C.c_void_p)
            call = lambda block: fn(entry, block)  # noqa: E731
        self.bound[bits] = call
        return call

    def __call__(self, bits, *args):
        """False when the arguments do not pack."""
        try:
            block = self.pack(*args)
        except struct.error:
            return False
        call = self.bound.get(bits) or self.bind(bits)
        if call(block):
            _check()
        return True


# ---- kernel entry points ---------------------------------------------------------------------
def _conv_like(name):
    packed = _Packed("conv", "=7Q16H2i", name)

    def call(bits, pInBuffer, pIm2ColBuffer, bias, pOutBuffer, pWeight, k, lambda_, out_mult,
             out_shift, dim_in_x, dim_in_y, ch_in, dim_out_x, dim_out_y, ch_out, dim_kernel_x,
             dim_kernel_y, padding_y_top, padding_y_bottom, padding_x_left, padding_x_right,
             stride_x, stride_y, flag_relu, flag_batch_norm):
        if packed(bits, _addr(pInBuffer), _addr(pIm2ColBuffer), _addr(bias), _addr(pOutBuffer), _addr(pWeight), _addr(k),
                  _addr(lambda_), out_mult, out_shift, dim_in_x, dim_in_y, ch_in, dim_out_x, dim_out_y, ch_out,
                  dim_kernel_x, dim_kernel_y, padding_y_top, padding_y_bottom, padding_x_left, padding_x_right, stride_x,
                  stride_y, flag_relu, flag_batch_norm):
            return
        _fn(name, bits)(_ptr(pInBuffer), _ptr(pIm2ColBuffer), _ptr(bias), _ptr(pOutBuffer),
                        _ptr(pWeight), _ptr(k), _ptr(lambda_), C.c_uint16(out_mult),
                        C.c_uint16(out_shift), C.c_uint16(dim_in_x), C.c_uint16(dim_in_y),
                        C.c_uint16(ch_in), C.c_uint16(dim_out_x), C.c_uint16(dim_out_y),
                        C.c_uint16(ch_out), C.c_uint16(dim_kernel_x), C.c_uint16(dim_kernel_y),
                        C.c_uint16(padding_y_top), C.c_uint16(padding_y_bottom),
                        C.c_uint16(padding_x_left), C.c_uint16(padding_x_right),
                        C.c_uint16(stride_x), C.c_uint16(stride_y), C.c_int(flag_relu),
                        C.c_int(flag_batch_norm))
        _check()
    call.__name__ = name
    call.__doc__ = "%s (32bit/include/pulp_nn_kernels.h); `bits` picks the tree." % name
    return call


pulp_nn_conv_Ho_parallel = _conv_like("pulp_nn_conv_Ho_parallel")
pulp_nn_conv_HoWo_parallel = _conv_like("pulp_nn_conv_HoWo_parallel")
pulp_nn_pointwise_HoWo_parallel = _conv_like("pulp_nn_pointwise_HoWo_parallel")
pulp_nn_conv_Co_parallel = _conv_like("pulp_nn_conv_Co_parallel")
pulp_nn_pointwise_Ho_parallel = _conv_like("pulp_nn_pointwise_Ho_parallel")
pulp_nn_pointwise_Co_parallel = _conv_like("pulp_nn_pointwise_Co_parallel")


def _dw_like(name):
    packed = _Packed("depthwise", "=8Q16H2b", name)

    def call(bits, Im_in, bufferC, bias, Im_out, wt, bufferB, k, lambda_, out_mult, out_shift,
             dim_im_in_x, dim_im_in_y, ch_im_in, dim_im_out_x, dim_im_out_y, ch_im_out,
             dim_kernel_x, dim_kernel_y, padding_y_top, padding_y_bottom, padding_x_left,
             padding_x_right, stride_x, stride_y, FLAG_RELU, FLAG_BATCH_NORM):
        if packed(bits, _addr(Im_in), _addr(bufferC), _addr(bias), _addr(Im_out), _addr(wt), _addr(bufferB), _addr(k),
                  _addr(lambda_), out_mult, out_shift, dim_im_in_x, dim_im_in_y, ch_im_in, dim_im_out_x, dim_im_out_y,
                  ch_im_out, dim_kernel_x, dim_kernel_y, padding_y_top, padding_y_bottom, padding_x_left, padding_x_right,
                  stride_x, stride_y, FLAG_RELU, FLAG_BATCH_NORM):
            return
        _fn(name, bits)(_ptr(Im_in), _ptr(bufferC), _ptr(bias), _ptr(Im_out), _ptr(wt),
                        _ptr(bufferB), _ptr(k), _ptr(lambda_), C.c_uint16(out_mult),
                        C.c_uint16(out_shift), C.c_uint16(dim_im_in_x), C.c_uint16(dim_im_in_y),
                        C.c_uint16(ch_im_in), C.c_uint16(dim_im_out_x), C.c_uint16(dim_im_out_y),
                        C.c_uint16(ch_im_out), C.c_uint16(dim_kernel_x), C.c_uint16(dim_kernel_y),
                        C.c_uint16(padding_y_top), C.c_uint16(padding_y_bottom),
                        C.c_uint16(padding_x_left), C.c_uint16(padding_x_right),
                        C.c_uint16(stride_x), C.c_uint16(stride_y), C.c_int8(FLAG_RELU),
                        C.c_int8(FLAG_BATCH_NORM))
        _check()
    call.__name__ = name
    return call


pulp_nn_depthwise_generic = _dw_like("pulp_nn_depthwise_generic")
pulp_nn_depthwise_generic_less_4_weights = _dw_like("pulp_nn_depthwise_generic_less_4_weights")
pulpnn_depthwise_hwc = _dw_like("pulpnn_depthwise_hwc")


def pulp_nn_depthwise_3x3_s1(bits, In_Img, Out_Img, R, C_, CH, p_l, p_r, Kernel, out_shift, out_mult, kappa,
                             lambda_, flag_relu, flag_batch_norm, memory_chan=None):
    """32bit/include/pulp_nn_kernels.h:340: CHW in (R x C), HWC out (R-2 x C), 3x3, stride 1."""
    _fn("pulp_nn_depthwise_3x3_s1", bits)(_ptr(In_Img), _ptr(Out_Img), C.c_int(R), C.c_int(C_), C.c_int(CH),
                                          C.c_int(p_l), C.c_int(p_r), _ptr(Kernel), C.c_int8(out_shift),
                                          C.c_uint16(out_mult), _ptr(kappa), _ptr(lambda_), C.c_int(flag_relu),
                                          C.c_int(flag_batch_norm), _ptr(memory_chan))
    _check()


def pulp_nn_matmul(bits, pWeight, pInBuffer, ch_out, num_col_im2col, out_shift, out_mult, k, lambda_, bias,
                   pOut, pOut2, flag_relu, flag_batch_norm):
    """32bit/include/pulp_nn_kernels.h:248. Returns the address the reference returns: pOut + 2*ch_out."""
    f = getattr(_lib.load_library(), "pulp_nn_matmul" + _sfx(bits))
    f.restype = C.c_void_p
    r = f(_ptr(pWeight), _ptr(pInBuffer), C.c_uint16(ch_out), C.c_uint16(num_col_im2col), C.c_uint16(out_shift),
          C.c_uint16(out_mult), _ptr(k), _ptr(lambda_), _ptr(bias), _ptr(pOut), _ptr(pOut2), C.c_int(flag_relu),
          C.c_int(flag_batch_norm))
    _check()
    return r


_linear = _Packed("linear", "=6QHb2H2i")
_linear_out_32 = _Packed("linear_out_32", "=4Q2H")
_maxpool = _Packed("maxpool", "=2Q13H")
_avgpool = _Packed("avgpool", "=2QqHq13Hi")
_add = _Packed("add", "=3Q6H")


def pulp_nn_linear(bits, pInBuffer, bias, pOutBuffer, pWeights, k, lambda_, out_mult, out_shift,
                   dim_vec, num_o_neurons, flag_relu, flag_batch_norm):
    if _linear(bits, _addr(pInBuffer), _addr(bias), _addr(pOutBuffer), _addr(pWeights), _addr(k), _addr(lambda_), out_mult,
               out_shift, dim_vec, num_o_neurons, flag_relu, flag_batch_norm):
        return
    _fn("pulp_nn_linear", bits)(_ptr(pInBuffer), _ptr(bias), _ptr(pOutBuffer), _ptr(pWeights),
                                _ptr(k), _ptr(lambda_), C.c_uint16(out_mult), C.c_int8(out_shift),
                                C.c_uint16(dim_vec), C.c_uint16(num_o_neurons), C.c_int(flag_relu),
                                C.c_int(flag_batch_norm))
    _check()


def pulp_nn_linear_out_32(bits, pInBuffer, bias, pOutBuffer, pWeights, dim_vec, num_o_neurons):
    if _linear_out_32(bits, _addr(pInBuffer), _addr(bias), _addr(pOutBuffer), _addr(pWeights), dim_vec, num_o_neurons):
        return
    _fn("pulp_nn_linear_out_32", bits)(_ptr(pInBuffer), _ptr(bias), _ptr(pOutBuffer),
                                       _ptr(pWeights), C.c_uint16(dim_vec),
                                       C.c_uint16(num_o_neurons))
    _check()


def _geom(dim_im_in_x, dim_im_in_y, ch_im_in, dim_im_out_x, dim_im_out_y, dim_kernel_x,
          dim_kernel_y, padding_t, padding_b, padding_l, padding_r, stride_x, stride_y):
    return [C.c_uint16(v) for v in (dim_im_in_x, dim_im_in_y, ch_im_in, dim_im_out_x, dim_im_out_y,
                                    dim_kernel_x, dim_kernel_y, padding_t, padding_b, padding_l,
                                    padding_r, stride_x, stride_y)]


def pulp_nn_maxpool(bits, Im_in, Im_out, dim_im_in_x, dim_im_in_y, ch_im_in, dim_im_out_x,
                    dim_im_out_y, dim_kernel_x, dim_kernel_y, padding_t, padding_b, padding_l,
                    padding_r, stride_x, stride_y):
    if _maxpool(bits, _addr(Im_in), _addr(Im_out), dim_im_in_x, dim_im_in_y, ch_im_in, dim_im_out_x, dim_im_out_y,
                dim_kernel_x, dim_kernel_y, padding_t, padding_b, padding_l, padding_r, stride_x, stride_y):
        return
    _fn("pulp_nn_maxpool", bits)(_ptr(Im_in), _ptr(Im_out),
                                 *_geom(dim_im_in_x, dim_im_in_y, ch_im_in, dim_im_out_x,
                                        dim_im_out_y, dim_kernel_x, dim_kernel_y, padding_t,
                                        padding_b, padding_l, padding_r, stride_x, stride_y))
    _check()


def pulp_nn_avgpool(bits, Im_in, Im_out, lambda_, out_shift, out_add, dim_im_in_x, dim_im_in_y,
                    ch_im_in, dim_im_out_x, dim_im_out_y, dim_kernel_x, dim_kernel_y, padding_t,
                    padding_b, padding_l, padding_r, stride_x, stride_y, flag_requant):
    if _avgpool(bits, _addr(Im_in), _addr(Im_out), int(lambda_), out_shift, int(out_add), dim_im_in_x, dim_im_in_y, ch_im_in,
                dim_im_out_x, dim_im_out_y, dim_kernel_x, dim_kernel_y, padding_t, padding_b, padding_l, padding_r,
                stride_x, stride_y, flag_requant):
        return
    bn_t = C.c_int32 if bits == 32 else C.c_int64
    _fn("pulp_nn_avgpool", bits)(_ptr(Im_in), _ptr(Im_out), bn_t(int(lambda_)),
                                 C.c_uint16(out_shift), bn_t(int(out_add)),
                                 *_geom(dim_im_in_x, dim_im_in_y, ch_im_in, dim_im_out_x,
                                        dim_im_out_y, dim_kernel_x, dim_kernel_y, padding_t,
                                        padding_b, padding_l, padding_r, stride_x, stride_y),
                                 C.c_int(flag_requant))
    _check()


def pulp_nn_add(bits, Im_in_1, Im_in_2, Im_out, out_mult1, out_mult2, out_shift, dim_im_in_h,
                dim_im_in_w, ch_im_in):
    if _add(bits, _addr(Im_in_1), _addr(Im_in_2), _addr(Im_out), out_mult1, out_mult2, out_shift, dim_im_in_h, dim_im_in_w,
            ch_im_in):
        return
    _fn("pulp_nn_add", bits)(_ptr(Im_in_1), _ptr(Im_in_2), _ptr(Im_out), C.c_uint16(out_mult1),
                             C.c_uint16(out_mult2), C.c_uint16(out_shift),
                             C.c_uint16(dim_im_in_h), C.c_uint16(dim_im_in_w),
                             C.c_uint16(ch_im_in))
    _check()


def _unpack(name):
    def call(src, dst, n_out):
        getattr(_lib.load_library(), name)(_ptr(src), _ptr(dst), C.c_uint(n_out))
        _check()
    call.__name__ = name
    call.__doc__ = "%s(src, dst, number of 8-bit results): sub-byte values widened to bytes." % name
    return call


pulp_nn_im2col_u4_to_u8 = _unpack("pulp_nn_im2col_u4_to_u8")
pulp_nn_im2col_u2_to_u8 = _unpack("pulp_nn_im2col_u2_to_u8")
pulpnn_i4_to_i8 = _unpack("pulpnn_i4_to_i8")
pulpnn_i2_to_i8 = _unpack("pulpnn_i2_to_i8")


def pulpnn_bn_quant_bulk(bits, phi, k, lambda_, d, out, n, channels, out_bits):
    """clip((k*phi + lambda) >> d) element-wise: pulp_nn_bn_quant_u8/u4/u2 in bulk; `bits` picks the tree."""
    getattr(_lib.load_library(), "pulpnn_bn_quant_bulk" + _sfx(bits))(
        _ptr(phi), _ptr(k), _ptr(lambda_), C.c_int8(d), _ptr(out), C.c_uint(n), C.c_uint(channels), C.c_int(out_bits))
    _check()


def pulpnn_quant_bulk(bits, phi, m, d, out, n, out_bits):
    """clip((m*phi) >> d) element-wise: pulp_nn_quant_u8/u4/u2 in bulk."""
    getattr(_lib.load_library(), "pulpnn_quant_bulk" + _sfx(bits))(
        _ptr(phi), C.c_int16(m), C.c_int8(d), _ptr(out), C.c_uint(n), C.c_int(out_bits))
    _check()


def pulpnn_threshold_quant_bulk(in_, thr, out, n, channels, out_bits):
    """pulp_nn_i4_quant / pulp_nn_i2_quant in bulk: thr is int16 [channels][16] (4 bits) or [channels][4] (2 bits)."""
    _lib.load_library().pulpnn_threshold_quant_bulk(_ptr(in_), _ptr(thr), _ptr(out), C.c_uint(n), C.c_uint(channels),
                                                    C.c_int(out_bits))
    _check()


def pulp_nn_avg_and_replace_int8(base, target, length):
    """32bit/include/pulp_nn_utils.h:39: base[i] = (base[i] + target[i]) >> 1 for length >> 2 whole words."""
    _lib.load_library().pulp_nn_avg_and_replace_int8(_ptr(base), _ptr(target), C.c_uint16(length))
    _check()


def pulpnn_chw_to_hwc(Im_in, Im_out, dim_im_x, dim_im_y, ch_im):
    """[batch][C][H][W] -> [batch][H][W][C] (no counterpart in the reference)."""
    _lib.load_library().pulpnn_chw_to_hwc(_ptr(Im_in), _ptr(Im_out), C.c_uint16(dim_im_x),
                                          C.c_uint16(dim_im_y), C.c_uint16(ch_im))
    _check()


def pulpnn_hwc_to_chw(Im_in, Im_out, dim_im_x, dim_im_y, ch_im):
    """[batch][H][W][C] -> [batch][C][H][W] (no counterpart in the reference)."""
    _lib.load_library().pulpnn_hwc_to_chw(_ptr(Im_in), _ptr(Im_out), C.c_uint16(dim_im_x),
                                          C.c_uint16(dim_im_y), C.c_uint16(ch_im))
    _check()


def pulpnn_linear_out_32_static_scratch(pInBuffer, bias, pOutBuffer, pWeights, dim_vec,
                                        num_o_neurons, n_vectors, k_slices):
    """pulp_nn_linear_out_32 arithmetic with split K for callers that may not allocate device
    memory: the partial sums go to a 4 MiB array built into the library instead of a buffer
    obtained with cudaMalloc. Device buffers only; k_slices * n_vectors * num_o_neurons must not
    exceed 1048576. Calls that overlap on the GPU share that array and race."""
    lib = _lib.load_library()
    rc = lib.pulpnn_linear_out_32_static_scratch(_ptr(pInBuffer), _ptr(bias), _ptr(pOutBuffer),
                                                 _ptr(pWeights), C.c_int(dim_vec),
                                                 C.c_int(num_o_neurons), C.c_int(n_vectors),
                                                 C.c_int(k_slices))
    if rc != OK:
        _check()
        raise PulpNNError(rc, "pulpnn_linear_out_32_static_scratch failed")


# ---- attention over a paged cache of keys and values ------------------------------------------
# The arguments go over as the C structs of include/pulpnn_b200.h, packed in one step; tensors are torch tensors on
# the context's GPU (anything with data_ptr, shape, stride and dtype). Shapes and types are checked here, alignment,
# ranges and whose memory it is by the library.
TYPE_F16, TYPE_BF16, TYPE_F32, TYPE_S32, TYPE_S8, TYPE_U8 = range(6)
_type_of = {}


def _type(x):
    code = _type_of.get(x.dtype)
    if code is None:
        if not _type_of:
            import torch
            _type_of.update({torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16, torch.float32: TYPE_F32,
                             torch.int32: TYPE_S32, torch.int8: TYPE_S8, torch.uint8: TYPE_U8, torch.int64: -2,
                             torch.float64: -3})
            return _type(x)
        raise PulpNNError(ERR_INVALID_ARG, "type %s" % x.dtype)
    return code


_TYPE_S64, _TYPE_F64 = -2, -3


def _need(ok, what):
    if not ok:
        raise PulpNNError(ERR_INVALID_ARG, what)


def _rows(x, name, n, heads, dim, type_, out=False):
    """Address, token and head stride of [n][heads][dim] rows; an axis of one has the stride 0."""
    a, b, c = x.stride()                  # of another rank: a ValueError, which the entry points turn into their error
    if x.shape != (n, heads, dim) or _type_of.get(x.dtype) != type_ or c != 1:
        raise PulpNNError(ERR_INVALID_ARG, "%s: %s %s with strides %s, where rows of %s are wanted" % (
            name, x.dtype, tuple(x.shape), x.stride(), (n, heads, dim)))
    a, b = a if n > 1 else 0, b if heads > 1 else 0
    if out and (a == 0 and n > 1 or b == 0 and heads > 1):
        raise PulpNNError(ERR_INVALID_ARG, "rows of %s share memory" % name)
    return x.data_ptr(), a, b


def _vector(x, name, n, type_):
    """Address of n contiguous values, 0 for None."""
    if x is None:
        return 0
    if x.numel() != n or _type_of.get(x.dtype) != type_ or not x.is_contiguous():
        raise PulpNNError(ERR_INVALID_ARG, "%s: %s %s, where %d values in one piece are wanted" % (name, x.dtype, tuple(x.shape), n))
    return x.data_ptr()


class _StructCall:
    """A C entry point that takes structs: call(struct, ...) raises what it records."""

    def __init__(self, name, n):
        self.name, self.n, self.f = name, n, None

    def __call__(self, *blocks):
        f = self.f
        if f is None:
            # the library's functions are shared objects of ctypes: a prototype of our own leaves theirs alone
            proto = C.CFUNCTYPE(C.c_int, *[C.c_char_p] * self.n)
            f = self.f = proto(C.cast(getattr(_lib.load_library(), self.name), C.c_void_p).value)
        if f(*blocks):
            _check()


# What unpacking a shape and packing a struct raise for tensors of another rank and numbers that the struct does not hold.
_MALFORMED = (struct.error, ValueError, IndexError, OverflowError)


def _malformed(name, e):
    return PulpNNError(ERR_INVALID_ARG, "%s: a tensor of another rank, or a number beyond its range (%s)" % (name, e))


class KVCache:
    """Pages of keys and values (pulpnn_kv_cache_t): k and v are [pages][slots][heads][dim], or [pages][heads][slots][dim]
    with heads_first, of type float16, bfloat16 or int8 with equal strides; int8 has k_scale and v_scale, float32
    without the last axis. The tensors stay the caller's, who keeps them on the GPU while calls use them."""

    _pack = struct.Struct("=4Q6q6i").pack

    def __init__(self, k, v, k_scale=None, v_scale=None, heads_first=False):
        shape, s, type_ = k.shape, k.stride(), _type(k)
        _need(len(shape) == 4 and v.shape == shape, "keys and values are of one shape, with four axes")
        _need(v.dtype == k.dtype and v.stride() == s, "keys and values are of one type, with the same strides")
        _need(s[3] == 1, "the channels of a row lie side by side")
        _need((s[0] or shape[0] == 1) and (s[1] or shape[1] == 1) and (s[2] or shape[2] == 1), "rows of the cache share memory")
        t = (0, 0, 0)
        if type_ == TYPE_S8:
            _need(k_scale is not None and v_scale is not None, "an int8 cache has scales")
            _need(k_scale.shape == shape[:3] and v_scale.shape == shape[:3], "scales are shaped as the cache without its last axis")
            _need(_type(k_scale) == TYPE_F32 and _type(v_scale) == TYPE_F32, "scales are float32")
            t = k_scale.stride()
            _need(v_scale.stride() == t, "scales have the same strides")
            _need((t[0] or shape[0] == 1) and (t[1] or shape[1] == 1) and (t[2] or shape[2] == 1), "scales share memory")
        else:
            _need(k_scale is None and v_scale is None, "a 16-bit cache has no scales")
        self.type, self.heads_first, self.tensors = type_, heads_first, (k, v, k_scale, v_scale)
        slot, head = (2, 1) if heads_first else (1, 2)          # the axes
        self.n_pages, self.page_size, self.n_heads, self.head_dim = shape[0], shape[slot], shape[head], shape[3]
        self.block = self._pack(k.data_ptr(), v.data_ptr(), _addr_of(k_scale), _addr_of(v_scale), s[0] if shape[0] > 1 else 0,
                                s[slot] if shape[slot] > 1 else 0, s[head] if shape[head] > 1 else 0, t[0], t[slot], t[head], type_,
                                self.n_pages, self.page_size, self.n_heads, self.head_dim, 0)


def _addr_of(x):
    return 0 if x is None else x.data_ptr()


_append_pack = struct.Struct("=12Q12q6i").pack
_append_call = _StructCall("pulpnn_kv_append", 2)
_gather_pack = struct.Struct("=3Q4q2i").pack
_gather_call = _StructCall("pulpnn_kv_gather", 2)


def pulpnn_kv_append(cache, slots, k, v, positions=None, inv_freq=None, interleaved=False, q=None, q_out=None, k_out=None,
                     v_out=None, q_step=None, k_step=None, v_step=None):
    """Rotates q and k ([tokens][heads][dim]; float16, bfloat16, float32, or int32 with a float32 step per channel) by
    positions (int32) x inv_freq (float64, half as many as channels rotate), writes q to q_out and stores k and v in the
    cache at slots (int64; one outside the cache stores nothing). k_out, v_out: the stored rows before a cut to 8 bits.
    The outputs are float16 or bfloat16, all of one type, which need not be the cache's."""
    try:
        n, heads, dim = k.shape[0], cache.n_heads, cache.head_dim
        if n == 0:
            return
        in_type = _type(k)
        o = q_out if q_out is not None else k_out if k_out is not None else v_out
        out_type = _type(o) if o is not None else cache.type if cache.type != TYPE_S8 else TYPE_BF16      # any, where no rows are written
        pk, pk0, pk1 = _rows(k, "k", n, heads, dim, in_type)
        pv, pv0, pv1 = _rows(v, "v", n, heads, dim, in_type)
        pq = pq0 = pq1 = oq = oq0 = oq1 = hq = ok = ok0 = ok1 = ov = ov0 = ov1 = sq = sk = sv = 0
        if q is not None:
            hq = q.shape[1]
            pq, pq0, pq1 = _rows(q, "q", n, hq, dim, in_type)
            _need(q_out is not None, "q and q_out come together")
            oq, oq0, oq1 = _rows(q_out, "q_out", n, hq, dim, out_type, True)
        elif q_out is not None:
            _need(False, "q and q_out come together")
        if k_out is not None:
            ok, ok0, ok1 = _rows(k_out, "k_out", n, heads, dim, out_type, True)
        if v_out is not None:
            ov, ov0, ov1 = _rows(v_out, "v_out", n, heads, dim, out_type, True)
        if in_type == TYPE_S32:
            _need(k_step is not None and v_step is not None and (q is None or q_step is not None), "int32 rows have steps")
            sq, sk, sv = (_vector(q_step, "q_step", hq * dim, TYPE_F32), _vector(k_step, "k_step", heads * dim, TYPE_F32),
                          _vector(v_step, "v_step", heads * dim, TYPE_F32))
        elif q_step is not None or k_step is not None or v_step is not None:
            _need(False, "steps are for int32 rows")
        at = angles = half = 0
        if inv_freq is not None:
            half = inv_freq.shape[0]
            _need(positions is not None or half == 0, "a rotation has positions")
            angles = _vector(inv_freq, "inv_freq", half, _TYPE_F64)
        if positions is not None:
            at = _vector(positions, "positions", n, TYPE_S32)
        _append_call(cache.block, _append_pack(
            pq, pk, pv, oq, ok, ov, sq, sk, sv, _vector(slots, "slots", n, _TYPE_S64), at, angles, pq0, pq1, pk0, pk1, pv0, pv1,
            oq0, oq1, ok0, ok1, ov0, ov1, n, hq, 2 * half, 1 if interleaved else 0, in_type, out_type))
    except _MALFORMED as e:
        raise _malformed("pulpnn_kv_append", e) from None


def pulpnn_kv_gather(cache, slots, k_out, v_out=None):
    """Rows `slots` (int64) of the cache into k_out and v_out ([tokens][heads][dim], float16 or bfloat16; either may be
    None). A slot outside the cache gives zeros."""
    try:
        n = slots.shape[0]
        if n == 0:
            return
        first = k_out if k_out is not None else v_out
        _need(first is not None, "neither k_out nor v_out")
        out_type, heads, dim = _type(first), cache.n_heads, cache.head_dim
        a = a0 = a1 = b = b0 = b1 = 0
        if k_out is not None:
            a, a0, a1 = _rows(k_out, "k_out", n, heads, dim, out_type, True)
        if v_out is not None:
            b, b0, b1 = _rows(v_out, "v_out", n, heads, dim, out_type, True)
        _gather_call(cache.block, _gather_pack(_vector(slots, "slots", n, _TYPE_S64), a, b, a0, a1, b0, b1, n, out_type))
    except _MALFORMED as e:
        raise _malformed("pulpnn_kv_gather", e) from None


_decode_pack = struct.Struct("=5Q5q2f8i").pack
_decode_call = _StructCall("pulpnn_attn_decode", 2)


def _out_type(out, in_type, out_step):
    """The type of an attention's output: the queries', or uint8 with a step."""
    type_ = _type(out)
    if type_ != in_type and type_ != TYPE_U8 or (type_ == TYPE_U8) != (out_step is not None):
        _need(False, "out is of q's type, or uint8; uint8 outputs, and only these, have an out_step")
    return type_


def pulpnn_attn_decode(cache, q, block_table, seq_lens, out, scale=None, window=0, lse=None, out_step=None, out_zero=0):
    """Attention of one new token per sequence: q and out [sequences][heads][dim], block_table int32 [sequences][pages],
    seq_lens int32 [sequences]. scale: dim ** -0.5 unless given. window > 0: the last `window` tokens only. lse: float32
    [sequences][heads]. out has q's type, or uint8 with out_step (and out_zero)."""
    try:
        n, heads, dim = q.shape
        if n == 0:
            return
        q_type = _type(q)
        out_type = _out_type(out, q_type, out_step)
        if dim != cache.head_dim:
            _need(False, "q and the cache have different numbers of channels")
        pq, q0, q1 = _rows(q, "q", n, heads, dim, q_type)
        po, o0, o1 = _rows(out, "out", n, heads, dim, out_type, True)
        shape, strides = block_table.shape, block_table.stride()
        if len(shape) != 2 or shape[0] != n or _type(block_table) != TYPE_S32 or (strides[1] != 1 and shape[1] > 1):
            _need(False, "block_table is int32 [sequences][pages], the pages of a sequence side by side")
        pages, lengths = shape[1], _vector(seq_lens, "seq_lens", n, TYPE_S32)
        _decode_call(cache.block, _decode_pack(
            pq, po, 0 if lse is None else _lse(lse, n, heads), block_table.data_ptr() if pages else lengths, lengths, q0, q1, o0, o1,
            strides[0] if n > 1 else 0, dim ** -0.5 if scale is None else scale, out_step or 0., out_zero, q_type, out_type, n, heads, pages,
            window, 0))
    except _MALFORMED as e:
        raise _malformed("pulpnn_attn_decode", e) from None


def _lse(lse, n, heads):
    _need(lse.shape == (n, heads) and lse.is_contiguous() and _type(lse) == TYPE_F32, "lse is float32 [rows][heads] in one piece")
    return lse.data_ptr()


_prompt_pack = struct.Struct("=7Q8q2f12i").pack
_prompt_call = _StructCall("pulpnn_attn_prompt", 1)


def pulpnn_attn_prompt(q, k, v, cu_q, out, cu_k=None, causal=True, window=0, scale=None, lse=None, out_step=None, out_zero=0):
    """Attention over whole prompts: sequence b holds rows cu_q[b] .. cu_q[b+1] of q and out ([rows][heads][dim]) and rows
    cu_k[b] .. cu_k[b+1] (cu_q's unless given) of k and v. Its last query and its last key have the same position.
    causal: no query sees a later position; window > 0 (causal only): nor one `window` or more before its own."""
    try:
        n, heads, dim = q.shape
        if n == 0:
            return
        nk, kv_heads = k.shape[0], k.shape[1]
        type_ = _type(q)
        out_type = _out_type(out, type_, out_step)
        pq, q0, q1 = _rows(q, "q", n, heads, dim, type_)
        pk, k0, k1 = _rows(k, "k", nk, kv_heads, dim, type_)
        pv, v0, v1 = _rows(v, "v", nk, kv_heads, dim, type_)
        po, o0, o1 = _rows(out, "out", n, heads, dim, out_type, True)
        seqs = cu_q.shape[0] - 1
        if cu_k is None:
            _need(nk == n, "other numbers of rows of keys than of queries, and no cu_k")
            cu_k = cu_q
        _prompt_call(_prompt_pack(
            pq, pk, pv, po, 0 if lse is None else _lse(lse, n, heads), _vector(cu_q, "cu_q", seqs + 1, TYPE_S32),
            _vector(cu_k, "cu_k", seqs + 1, TYPE_S32), q0, q1, k0, k1, v0, v1, o0, o1, dim ** -0.5 if scale is None else scale,
            out_step or 0., out_zero, type_, out_type, n, nk, seqs, heads, kv_heads, dim, 1 if causal else 0, window, 0))
    except _MALFORMED as e:
        raise _malformed("pulpnn_attn_prompt", e) from None


# ---- network runner --------------------------------------------------------------------------
class LayerDesc(C.Structure):
    _fields_ = [(n, C.c_int) for n in (
        "type", "dim_in_x", "dim_in_y", "ch_in", "dim_out_x", "dim_out_y", "ch_out",
        "dim_kernel_x", "dim_kernel_y", "padding_y_top", "padding_y_bottom", "padding_x_left",
        "padding_x_right", "stride_x", "stride_y", "out_mult", "out_shift", "flag_relu",
        "flag_batch_norm")] + [("weights", C.c_void_p), ("bias", C.c_void_p), ("k", C.c_void_p),
                               ("lambda_", C.c_void_p)]


class Net:
    """Sequential network on one GPU (pulpnn_net_* in include/pulpnn_b200.h)."""

    def __init__(self, bits, max_batch):
        self.lib = _lib.load_library()
        self.bits = bits
        self.max_batch = max_batch
        self.handle = self.lib.pulpnn_net_create(int(bits), int(max_batch))
        if not self.handle:
            _check()
            raise PulpNNError(ERR_CUDA, "pulpnn_net_create failed")
        self.handle = C.c_void_p(self.handle)

    def add_layer(self, type_, *, dim_in, ch_in, dim_out, ch_out, kernel=(1, 1), pads=(0, 0, 0, 0),
                  strides=(1, 1), out_mult=1, out_shift=0, relu=1, bn=1, weights=None, bias=None,
                  k=None, lam=None):
        d = LayerDesc()
        d.type = type_
        d.dim_in_y, d.dim_in_x = dim_in
        d.ch_in = ch_in
        d.dim_out_y, d.dim_out_x = dim_out
        d.ch_out = ch_out
        d.dim_kernel_y, d.dim_kernel_x = kernel
        d.padding_y_top, d.padding_y_bottom, d.padding_x_left, d.padding_x_right = pads
        d.stride_y, d.stride_x = strides
        d.out_mult, d.out_shift, d.flag_relu, d.flag_batch_norm = out_mult, out_shift, relu, bn
        for name, arr in (("weights", weights), ("bias", bias), ("k", k), ("lambda_", lam)):
            p = _ptr(arr)
            setattr(d, name, p.value if p is not None else None)
        if self.lib.pulpnn_net_add_layer(self.handle, C.byref(d)) != OK:
            _check()

    def finalize(self, micro_batch=0):
        if self.lib.pulpnn_net_finalize(self.handle, int(micro_batch)) != OK:
            _check()

    def run(self, input_, output, n_images, n_layers=None):
        if n_layers is None:
            rc = self.lib.pulpnn_net_run(self.handle, _ptr(input_), _ptr(output), int(n_images))
        else:
            rc = self.lib.pulpnn_net_run_prefix(self.handle, _ptr(input_), _ptr(output),
                                                int(n_images), int(n_layers))
        if rc != OK:
            _check()

    def submit(self, input_, output, n_images):
        """Host buffers, no waiting: returns a ticket for wait(). Two batches may be in flight."""
        t = self.lib.pulpnn_net_submit(self.handle, _ptr(input_), _ptr(output), int(n_images))
        if t < 0:
            _check()
            raise PulpNNError(-t, "pulpnn_net_submit failed")
        return t

    def wait(self, ticket):
        if self.lib.pulpnn_net_wait(self.handle, int(ticket)) != OK:
            _check()

    def run_timed(self, input_, output, n_images):
        """Device buffers only. Returns the per-layer milliseconds of this run."""
        ms = (C.c_float * self.num_layers())()
        if self.lib.pulpnn_net_run_timed(self.handle, _ptr(input_), _ptr(output), int(n_images), ms) != OK:
            _check()
        return list(ms)

    def num_layers(self):
        return self.lib.pulpnn_net_num_layers(self.handle)

    def layer_role(self, layer):
        """0: own kernel; 1 / 2: first / second layer of a fused pair (in the most recent run)."""
        return int(self.lib.pulpnn_net_layer_role(self.handle, int(layer)))

    def layer_kernel(self, layer):
        """Kernel family that ran the layer in the most recent run."""
        return (self.lib.pulpnn_net_layer_kernel(self.handle, int(layer)) or b"").decode()

    def layer_output_bytes(self, layer):
        return int(self.lib.pulpnn_net_layer_output_bytes(self.handle, int(layer)))

    def close(self):
        if self.handle:
            self.lib.pulpnn_net_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def build_mobilenet_v1(params, bits=32, max_batch=1024, micro_batch=0):
    """MobileNetV1 as a Net from workloads.mobilenet_params(): conv1, 13 x (depthwise, pointwise),
    global average pool, fully connected layer with int32 logits."""
    net = Net(bits, max_batch)
    dt = np.int32 if bits == 32 else np.int64
    for p in params:
        common = dict(dim_in=(p["H"], p["W"]), ch_in=p["Cin"], dim_out=(p["Ho"], p["Wo"]),
                      ch_out=p["Cout"])
        if p["op"] == "conv":
            net.add_layer(LAYER_CONV, kernel=(3, 3), pads=(1, 1, 1, 1),
                          strides=(p["stride"], p["stride"]), out_shift=p["out_shift"],
                          weights=p["w"], k=np.ascontiguousarray(p["k"], dt),
                          lam=np.ascontiguousarray(p["lam"], dt), **common)
        elif p["op"] == "depthwise":
            net.add_layer(LAYER_DEPTHWISE, kernel=(3, 3), pads=(1, 1, 1, 1),
                          strides=(p["stride"], p["stride"]), out_shift=p["out_shift"],
                          weights=p["w"], k=np.ascontiguousarray(p["k"], dt),
                          lam=np.ascontiguousarray(p["lam"], dt), **common)
        elif p["op"] == "pointwise":
            net.add_layer(LAYER_POINTWISE, out_shift=p["out_shift"], weights=p["w"],
                          k=np.ascontiguousarray(p["k"], dt),
                          lam=np.ascontiguousarray(p["lam"], dt), **common)
        elif p["op"] == "avgpool":
            net.add_layer(LAYER_AVGPOOL, kernel=(p["H"], p["W"]), strides=(p["H"], p["W"]), **common)
        elif p["op"] == "linear32":
            net.add_layer(LAYER_LINEAR_OUT_32, weights=p["w"], **common)
        else:
            raise ValueError(p["op"])
    net.finalize(micro_batch)
    return net
