// The mixture-of-experts layer on int8 weights of the CUDA backend (og_int8_moe_*). No counterpart in the reference.
using RecursiveAI.OneGpu.Kernels;

namespace RecursiveAI.OneGpu.Cuda;

/// <summary>A layer for up to 128 tokens, offsets in elements. Gated: hidden values are activation(first half) * second
/// half of an expert's input product. Normalize: the chosen experts' weights sum to one.</summary>
public struct MoeProblem
{
    public int Tokens, ModelSize, ExpertSize, Experts, TopK;
    public Int8Activation Activation = Int8Activation.Silu;
    public bool Gated = true, Normalize = true;
    public int OffsetX, OffsetRouter, OffsetIn, OffsetInScale, OffsetOut, OffsetOutScale, OffsetY;
    public int OffsetResidual, OffsetIds, OffsetWeights;

    // Without it `new MoeProblem { .. }` would skip the initializers above.
    public MoeProblem() { }

    public MoeProblem(int tokens, int modelSize, int expertSize, int experts, int topK)
    {
        Tokens = tokens;
        ModelSize = modelSize;
        ExpertSize = expertSize;
        Experts = experts;
        TopK = topK;
    }

    internal readonly OgMoeProblem Native() => new()
    {
        Tokens = Tokens, ModelSize = ModelSize, ExpertSize = ExpertSize, Experts = Experts, TopK = TopK,
        Activation = (int)Activation, Gated = Gated ? 1 : 0, Normalize = Normalize ? 1 : 0,
        OffsetX = OffsetX, OffsetRouter = OffsetRouter, OffsetIn = OffsetIn, OffsetInScale = OffsetInScale,
        OffsetOut = OffsetOut, OffsetOutScale = OffsetOutScale, OffsetY = OffsetY, OffsetResidual = OffsetResidual,
        OffsetIds = OffsetIds, OffsetWeights = OffsetWeights,
    };
}

/// <summary>A whole mixture-of-experts layer for a few tokens: the router, the choice of each token's experts, their
/// feed-forward products on int8 weights and the weighted sum. Not thread-safe.</summary>
public sealed unsafe class Int8MoeKernels : IDisposable
{
    nint _handle;

    public Int8MoeKernels(GpuDevice device)
    {
        ArgumentNullException.ThrowIfNull(device);
        if (device is not CudaDevice cuda)
            throw new GpuUnsupportedException("Int8MoeKernels of the CUDA backend needs a CUDA device", "Backend", "CUDA",
                                              device.Backend.ToString());
        nint h;
        NativeCheck.Check(Cuda.Native.og_int8_moe_create(cuda.Handle, &h));
        _handle = h;
    }

    nint Handle => _handle != 0 ? _handle : throw new ObjectDisposedException(nameof(Int8MoeKernels));

    /// <summary>y = residual + sum over a token's experts of w * (expert's feed-forward of x); T is float or Half, TR the
    /// router's type; expertIds and expertWeights receive the routing.</summary>
    public void Encode<T, TR>(GpuCommandEncoder encoder, in MoeProblem problem, GpuBuffer<T> x, GpuBuffer<TR> router,
                              GpuBuffer<sbyte> wIn, GpuBuffer<float> wInScale, GpuBuffer<sbyte> wOut,
                              GpuBuffer<float> wOutScale, GpuBuffer<T> y, GpuBuffer<T>? residual = null,
                              GpuBuffer<int>? expertIds = null, GpuBuffer<float>? expertWeights = null)
        where T : unmanaged
        where TR : unmanaged
    {
        ArgumentNullException.ThrowIfNull(encoder);
        var enc = encoder as CudaCommandEncoder
                  ?? throw new GpuUnsupportedException("the encoder belongs to another backend", "Backend", "CUDA", null);
        var p = problem.Native();
        OgBuffer vx = NativeCheck.View(x), vr = NativeCheck.View(router), vi = NativeCheck.View(wIn);
        OgBuffer vis = NativeCheck.View(wInScale), vo = NativeCheck.View(wOut), vos = NativeCheck.View(wOutScale);
        OgBuffer vy = NativeCheck.View(y), vres = NativeCheck.View(residual), vid = NativeCheck.View(expertIds);
        OgBuffer vw = NativeCheck.View(expertWeights);
        NativeCheck.Check(Cuda.Native.og_int8_moe_encode(Handle, enc.Handle, &p, &vx, &vr, &vi, &vis, &vo, &vos, &vy,
                                                         residual is null ? null : &vres,
                                                         expertIds is null ? null : &vid,
                                                         expertWeights is null ? null : &vw));
    }

    public void Dispose()
    {
        if (_handle == 0) return;
        Cuda.Native.og_int8_moe_destroy(_handle);
        _handle = 0;
    }
}
