# B200Backend.jl — the reference-side binding of libb200dnn.so.
#
# Drop this file into DNNKernels/src and `include("B200Backend.jl")` after kernelplans.jl.
# It adds a backend, a device array, the caps answer, new plan types and one method per
# entry point (`matmul!`, `sdpa!`, `layernorm!`, `convolution!`, `scratch!`, `toback`), which is
# the extension rule the package states: a new path is a new plan type plus a new method
# (kernels/extern/matmul.jl:97-100, kernels/extern/attention.jl:767-771, kernelplans.jl:1-19).
# Nothing else in the package changes: `execute!`, the rewrite passes, `planslab` and `dest`
# keep working because `B200Array` is a dense column-major array like `LavaArray`.
#
# No Julia toolchain exists where this file was written, so it has not been executed; the
# identical call sequence is exercised through the same C symbols by the Python mirror in
# juliavision_b200/*.py and its tests.

module B200

using ..DNNKernels: Ctx, Decline, MMGemvPlan, accum, actfn, geluexact, gelutanh, relu_epi
import ..DNNKernels: matmul!, mmplan, mm_gemv_plan, batchedmatmul!, sdpa!, sdpaplan, layernorm!, convolution!,
                     maxpool2d!, scratch!, toback, caps, slabview
import KernelAbstractions

const LIB = get(ENV, "B200DNN_LIB", "libb200dnn.so")

# ------------------------------------------------------------------ status handling
const OK = Cint(0)
const DECLINE = Dict(16 => :operands, 17 => :extent, 18 => :wrapped, 19 => :bias, 20 => :eltype, 21 => :tiling)
lasterror() = unsafe_string(ccall((:b200_last_error, LIB), Cstring, ()))
check(rc::Cint) = rc == OK ? nothing : error("b200dnn status $rc: $(lasterror())")

# ------------------------------------------------------------------ backend / arrays
mutable struct B200Backend <: KernelAbstractions.GPU
    handle::Ptr{Cvoid}
    device::Int
    function B200Backend(device::Integer = 0)
        h = Ref{Ptr{Cvoid}}(C_NULL)
        check(ccall((:b200_ctx_create, LIB), Cint, (Cint, Ref{Ptr{Cvoid}}), device, h))
        b = new(h[], device)
        finalizer(x -> ccall((:b200_ctx_destroy, LIB), Cint, (Ptr{Cvoid},), x.handle), b)
    end
end

"""Dense column-major device array; `parent` keeps the pool block or slab alive."""
struct B200Array{T,N} <: DenseArray{T,N}
    ptr::Ptr{T}
    dims::NTuple{N,Int}
    backend::B200Backend
    parent::Any
end
Base.size(a::B200Array) = a.dims
Base.pointer(a::B200Array) = a.ptr
Base.strides(a::B200Array) = Base.size_to_strides(1, a.dims...)
KernelAbstractions.get_backend(a::B200Array) = a.backend
KernelAbstractions.synchronize(b::B200Backend) = check(ccall((:b200_sync, LIB), Cint, (Ptr{Cvoid},), b.handle))

mutable struct PoolBlock
    backend::B200Backend
    ptr::Ptr{Cvoid}
end
function KernelAbstractions.allocate(b::B200Backend, ::Type{T}, dims::Integer...) where {T}
    p = Ref{Ptr{Cvoid}}(C_NULL)
    check(ccall((:b200_pool_alloc, LIB), Cint, (Ptr{Cvoid}, Csize_t, Ref{Ptr{Cvoid}}), b.handle,
                max(prod(dims), 1) * sizeof(T), p))
    blk = PoolBlock(b, p[])
    finalizer(x -> ccall((:b200_pool_free, LIB), Cint, (Ptr{Cvoid}, Ptr{Cvoid}), x.backend.handle, x.ptr), blk)
    B200Array{T,length(dims)}(Ptr{T}(p[]), Int.(dims), b, blk)
end

"""`toback(backend, a)` (driver.jl:108-115): upload a host array."""
function toback(b::B200Backend, a::AbstractArray{T}) where {T}
    h = Array(a)
    d = KernelAbstractions.allocate(b, T, size(h)...)
    check(ccall((:b200_upload, LIB), Cint, (Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Csize_t), b.handle, d.ptr, h,
                sizeof(h)))
    d
end
function Base.Array(a::B200Array{T,N}) where {T,N}
    h = Array{T,N}(undef, a.dims)
    check(ccall((:b200_download, LIB), Cint, (Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Csize_t), a.backend.handle, h,
                a.ptr, sizeof(h)))
    h
end

"""`slabview(T, slab, dims, off)` (execute.jl:173-179): a typed view at a byte offset of a slab."""
slabview(::Type{T}, slab::B200Array{UInt8,1}, dims, off::Integer) where {T} =
    B200Array{T,length(dims)}(Ptr{T}(slab.ptr + off), Int.(Tuple(dims)), slab.backend, slab)

"""`scratch!(ws, backend, T, dims...)` (workspace.jl:63-96) served by the library's bump workspace."""
function scratch!(::Any, b::B200Backend, ::Type{T}, dims::Integer...) where {T}
    p = Ref{Ptr{Cvoid}}(C_NULL)
    check(ccall((:b200_workspace_scratch, LIB), Cint, (Ptr{Cvoid}, Csize_t, Ref{Ptr{Cvoid}}), b.handle,
                prod(dims) * sizeof(T), p))
    B200Array{T,length(dims)}(Ptr{T}(p[]), Int.(dims), b, nothing)
end
resetworkspace!(b::B200Backend) = check(ccall((:b200_workspace_reset, LIB), Cint, (Ptr{Cvoid},), b.handle))

# ------------------------------------------------------------------ caps (context.jl:55-68)
struct CapsC
    coopmat::Int32; tile::Int32; subgroup::Int32; coopmatsubgroup::Int32; sharedbudget::Int32
    workgrouplimit::Int32; cores::Int32; warps::Int32; cc_major::Int32; cc_minor::Int32; total_mem::Int64
end
struct B200Caps
    coopmat::Bool; tile::Int; subgroup::Int; coopmatsubgroup::Int; sharedbudget::Int
    workgrouplimit::Int; cores::Int; warps::Int
end
function caps(b::B200Backend)
    c = Ref{CapsC}()
    check(ccall((:b200_caps, LIB), Cint, (Ptr{Cvoid}, Ref{CapsC}), b.handle, c))
    B200Caps(c[].coopmat != 0, c[].tile, c[].subgroup, c[].coopmatsubgroup, c[].sharedbudget,
             c[].workgrouplimit, c[].cores, c[].warps)
end

# ------------------------------------------------------------------ plans
"""Tensor-core GEMM plan; no padded extent — ragged M/N/K are TMA-clipped tiles."""
struct MMTilePlan end
"""fp16 operands a tensor map cannot express: the scalar kernel (mm2's arithmetic) on the GPU."""
struct MMScalarPlan end
"""Fused single-pass attention on tcgen05."""
struct FlashTCPlan end
struct AttnScalarPlan end
struct TwoGemmPlan end     # head dims above 128 (multiples of 8): the two-GEMM route inside the library

dtcode(::Type{Float16}) = Cint(0)
dtcode(::Type{Float32}) = Cint(1)
epicode(epi) = epi === geluexact ? Cint(2) : epi === relu_epi ? Cint(1) : epi === gelutanh ? Cint(3) :
               epi === identity ? Cint(0) : error("no fused form for epilogue $epi")

"""Root pointer + strides of a wrapper stack over a B200Array (the job of `stridedroot`,
attention.jl:321-337): `nothing` when the stack is not a strided view."""
function rootstrides(a)
    a isa B200Array && return (pointer(a), strides(a))
    try
        return (pointer(a), strides(a))     # SubArray / PermutedDimsArray / ReshapedArray of dense parents
    catch
        return nothing
    end
end

# ------------------------------------------------------------------ matmul! (matmul.jl:78-100)
function mmplan(dev::B200Caps, out, A, B, bias)
    if size(B, 2) == 1                       # one token: the matrix-vector kernel (fp32 as in the reference, or fp16)
        g = mm_gemv_plan(dev, out, A, B, bias)
        g isa MMGemvPlan && return g
    end
    eltype(A) === Float16 && eltype(B) === Float16 || return Decline(:operands)
    eltype(out) in (Float16, Float32) || return Decline(:eltype)
    ra, rb, ro = rootstrides(A), rootstrides(B), rootstrides(out)
    (ra === nothing || rb === nothing || ro === nothing) && return Decline(:wrapped)
    (ra[2][1] == 1 && rb[2][1] == 1 && ro[2][1] == 1) || return Decline(:wrapped)
    M, K = size(A); N = size(B, 2)
    rc = ccall((:b200_gemm_f16_supported, LIB), Cint, (Int64, Int64, Int64, Int64, Int64, Int64, Cint),
               M, N, K, ra[2][2], rb[2][2], ro[2][2], dtcode(eltype(out)))
    rc == OK && return MMTilePlan()
    rc == 18 && return MMScalarPlan()
    Decline(get(DECLINE, Int(rc), :extent))
end

function matmul!(ctx, ::Union{MMTilePlan,MMScalarPlan}, out, A, B, bias, epi; gemm = NamedTuple())
    M, K = size(A); N = size(B, 2)
    check(ccall((:b200_gemm_f16, LIB), Cint,
                (Ptr{Cvoid}, Int64, Int64, Int64, Ptr{Cvoid}, Int64, Ptr{Cvoid}, Int64, Ptr{Cvoid}, Ptr{Cvoid},
                 Int64, Cint, Cint, Int64, Int64, Int64, Int64),
                ctx.backend.handle, M, N, K, pointer(A), stride(A, 2), pointer(B), stride(B, 2),
                bias === nothing ? C_NULL : pointer(bias), pointer(out), stride(out, 2), dtcode(eltype(out)),
                epicode(epi), 1, 0, 0, 0))
    out
end
# No CPU path behind this backend: a refusal is an error, not a slower route.
matmul!(ctx::Ctx{B200Backend}, d::Decline, out, A, B, bias, epi; gemm = NamedTuple()) =
    error("matmul!: Decline(:$(d.reason)) on the B200 backend")

function batchedmatmul!(ctx::Ctx{B200Backend}, out, A, B)
    M, K, nb = size(A); N = size(B, 2)
    check(ccall((:b200_gemm_f16, LIB), Cint,
                (Ptr{Cvoid}, Int64, Int64, Int64, Ptr{Cvoid}, Int64, Ptr{Cvoid}, Int64, Ptr{Cvoid}, Ptr{Cvoid},
                 Int64, Cint, Cint, Int64, Int64, Int64, Int64),
                ctx.backend.handle, M, N, K, pointer(A), stride(A, 2), pointer(B), stride(B, 2), C_NULL,
                pointer(out), stride(out, 2), dtcode(eltype(out)), 0, nb, stride(A, 3), stride(B, 3),
                stride(out, 3)))
    out
end

# ------------------------------------------------------------------ sdpa! (attention.jl:712-834)
struct Strided4
    ptr::Ptr{Cvoid}
    stride::NTuple{4,Int64}
end
s4(a) = (r = rootstrides(a); Strided4(Ptr{Cvoid}(r[1]), Int64.(r[2])))

# An additive mask does not decline here: the fused kernel adds it (b200_attention_f16_bias).  It must
# be Float16 and broadcast to (Lk, Lq, H, B), the graph's own order (attention.jl:55-59).
function sdpaplan(ctx::Ctx{B200Backend}, q, k, v, bias)
    if bias !== nothing
        eltype(bias) === Float16 || return (Decline(:eltype), k, v)
        all(i -> size(bias, i) in (1, (size(k, 2), size(q, 2), size(q, 3), size(q, 4))[i]), 1:4) ||
            return (Decline(:bias), k, v)
    end
    all(x -> eltype(x) === Float16, (q, k, v)) || return (Decline(:eltype), k, v)
    any(x -> rootstrides(x) === nothing, (q, k, v)) && return (Decline(:wrapped), k, v)
    E, Lq, H, B = size(q); Lk = size(k, 2)
    st(x) = collect(Int64.(rootstrides(x)[2]))
    rc = ccall((:b200_attention_f16_supported, LIB), Cint,
               (Int64, Int64, Int64, Int64, Int64, Ptr{Int64}, Ptr{Int64}, Ptr{Int64}, Cint),
               E, Lq, Lk, H, B, st(q), st(k), st(v), 0)
    rc == OK && return (FlashTCPlan(), k, v)
    if rc in (18, 21)
        # head dims above 128: S = K'Q, softmax over the keys, O = V P on the GEMM kernel (route 1), else scalar
        route = ccall((:b200_attention_f16_route, LIB), Cint,
                      (Int64, Int64, Int64, Int64, Int64, Ptr{Int64}, Ptr{Int64}, Ptr{Int64}),
                      E, Lq, Lk, H, B, st(q), st(k), st(v))
        return (route == 1 ? TwoGemmPlan() : AttnScalarPlan(), k, v)
    end
    (Decline(get(DECLINE, Int(rc), :extent)), k, v)
end

function sdpa!(ctx, ::Union{FlashTCPlan,TwoGemmPlan,AttnScalarPlan}, out, q, k, v, bias, scale)
    E, Lq, H, B = size(q); Lk = size(k, 2)
    out === nothing && (out = KernelAbstractions.allocate(ctx.backend, accum(eltype(q)), E, Lq, H, B))
    # `out` may be any (E, Lq, H, B) view with E contiguous: a token-major destination folds the
    # clone that follows sdpa in the exported graphs into the store.
    if bias === nothing
        check(ccall((:b200_attention_f16_strided, LIB), Cint,
                    (Ptr{Cvoid}, Int64, Int64, Int64, Int64, Int64, Ref{Strided4}, Ref{Strided4}, Ref{Strided4},
                     Ref{Strided4}, Cint, Cfloat),
                    ctx.backend.handle, E, Lq, Lk, H, B, s4(q), s4(k), s4(v), s4(out), dtcode(eltype(out)),
                    Float32(scale)))
    else
        b = s4(bias)   # a size-1 axis broadcasts: stride 0
        b = Strided4(b.ptr, ntuple(i -> size(bias, i) == 1 ? Int64(0) : b.stride[i], 4))
        check(ccall((:b200_attention_f16_bias, LIB), Cint,
                    (Ptr{Cvoid}, Int64, Int64, Int64, Int64, Int64, Ref{Strided4}, Ref{Strided4}, Ref{Strided4},
                     Ref{Strided4}, Ref{Strided4}, Cint, Cfloat),
                    ctx.backend.handle, E, Lq, Lk, H, B, s4(q), s4(k), s4(v), b, s4(out), dtcode(eltype(out)),
                    Float32(scale)))
    end
    out
end

# ------------------------------------------------------------------ layernorm! (layernorm.jl:125-135)
function layernorm!(ctx::Ctx{B200Backend}, out, mean, rstd, a, γ, β, C::Integer, eps::Real)
    groups = length(a) ÷ C
    check(ccall((:b200_layernorm, LIB), Cint,
                (Ptr{Cvoid}, Int64, Int64, Ptr{Cvoid}, Cint, Ptr{Cvoid}, Cint, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid},
                 Ptr{Cvoid}, Cfloat),
                ctx.backend.handle, groups, C, pointer(a), dtcode(eltype(a)), pointer(out), dtcode(eltype(out)),
                pointer(mean), pointer(rstd), γ === nothing ? C_NULL : pointer(γ),
                β === nothing ? C_NULL : pointer(β), Float32(eps)))
    out
end

# x .= clamp.(x .+ h); layernorm!(out, mean, rstd, x, ...) in one launch: the target of a load-time
# rewrite that folds add.Tensor (+ clamp.default) into the native_layer_norm that follows.
function addlayernorm!(ctx::Ctx{B200Backend}, out, mean, rstd, x, h, γ, β, C::Integer, eps::Real; clamp = nothing)
    lo, hi = clamp === nothing ? (0f0, 0f0) : Float32.(clamp)
    check(ccall((:b200_add_layernorm_f16, LIB), Cint,
                (Ptr{Cvoid}, Int64, Int64, Ptr{Cvoid}, Ptr{Cvoid}, Cint, Cfloat, Cfloat, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid},
                 Ptr{Cvoid}, Ptr{Cvoid}, Cfloat),
                ctx.backend.handle, length(x) ÷ C, C, pointer(x), pointer(h), clamp === nothing ? 0 : 1, lo, hi,
                pointer(out), pointer(mean), pointer(rstd), γ === nothing ? C_NULL : pointer(γ),
                β === nothing ? C_NULL : pointer(β), Float32(eps)))
    out
end

# ------------------------------------------------------------------ matmul!(::MMGemvPlan) (matmul.jl:103-137)
function mm_gemv_plan(dev::B200Caps, out, A, B, bias)
    T = eltype(A)
    (T === Float32 || T === Float16) && eltype(B) === T || return Decline(:operands)
    size(B, 2) == 1 || return Decline(:notvector)
    bias === nothing || (bias isa AbstractVector && length(bias) == size(A, 1)) || return Decline(:bias)
    MMGemvPlan()
end
function matmul!(ctx::Ctx{B200Backend}, ::MMGemvPlan, out, A, B, bias, epi; gemm = NamedTuple())
    M, K = size(A)
    check(ccall((:b200_gemv, LIB), Cint,
                (Ptr{Cvoid}, Int64, Int64, Ptr{Cvoid}, Int64, Ptr{Cvoid}, Ptr{Cvoid}, Cint, Ptr{Cvoid}, Cint, Cint),
                ctx.backend.handle, M, K, pointer(A), stride(A, 2), pointer(B),
                bias === nothing ? C_NULL : pointer(bias), dtcode(eltype(A)), pointer(out), dtcode(eltype(out)),
                epicode(epi)))
    out
end

# ------------------------------------------------------------------ a decoder's step (new surface)
# Counts (`lens`, `news`, `starts`) are Int32 device vectors of one number a sequence; rows are (E, L, H, B) views, E contiguous.
nullable(a) = a === nothing ? C_NULL : pointer(a)

# freq: `rot ÷ 2` UInt64 on the device, radians a position / 2π modulo one, in units of 2^-64.
struct RotaryPlan
    rot::Int64
    interleaved::Bool
    gain::Float32
    freq::B200Array{UInt64,1}
end
function rotary!(ctx::Ctx{B200Backend}, plan::RotaryPlan, out, x; lens, news = nothing)
    E, L, H, B = size(x)
    check(ccall((:b200_rotary_f16, LIB), Cint,
                (Ptr{Cvoid}, Int64, Int64, Int64, Int64, Ref{Strided4}, Ref{Strided4}, Ptr{Cvoid}, Int64, Cint, Cfloat,
                 Ptr{Cvoid}, Int64, Int64, Ptr{Cvoid}, Ptr{Cvoid}),
                ctx.backend.handle, E, L, H, B, s4(x), s4(out), pointer(plan.freq), plan.rot, plan.interleaved, plan.gain,
                C_NULL, 0, 0, pointer(lens), nullable(news)))
    out
end

# The library sees pointers and the sizes it is told: what they are taken from is compared first.
demand(ok, what) = ok || throw(DimensionMismatch(what))
dense(a) = strides(a) == Base.size_to_strides(1, size(a)...)
isdense(a, T, dims...) = eltype(a) === T && size(a) == dims && dense(a)
iscounts(a, n) = a === nothing || (eltype(a) === Int32 && length(a) == n && dense(a))
along(a) = size(a, 1) <= 1 || stride(a, 1) == 1

# weight (E,), (E, H), or with split (E, 2): heads up to `split` take its first column.
function normrotary!(ctx::Ctx{B200Backend}, plan::RotaryPlan, out, x, weight = nothing; eps = 1f-6, split = nothing, lens, news = nothing)
    demand(ndims(x) == 4 && eltype(x) === eltype(out) === Float16 && size(out) == size(x), "normrotary!: x and out are (E, L, H, B) of Float16")
    E, L, H, B = size(x)
    demand(lens !== nothing && iscounts(lens, B) && iscounts(news, B), "normrotary!: lens and news are one Int32 a sequence")
    demand(2 * length(plan.freq) >= plan.rot, "normrotary!: the plan has a frequency for each pair")
    demand(split === nothing || (weight !== nothing && 0 <= split <= H), "normrotary!: split between the heads of a weight")
    demand(weight === nothing || (eltype(weight) in (Float16, Float32) && ndims(weight) in (1, 2) && size(weight, 1) == E && along(weight) &&
                                  (split === nothing ? size(weight, 2) in (1, H) : size(weight, 2) == 2)),
           "normrotary!: weight is (E,), (E, H), or with split (E, 2)")
    check(ccall((:b200_norm_rotary_f16, LIB), Cint,
                (Ptr{Cvoid}, Int64, Int64, Int64, Int64, Ref{Strided4}, Ref{Strided4}, Ptr{Cvoid}, Cint, Int64, Int64, Cfloat,
                 Ptr{Cvoid}, Int64, Cint, Cfloat, Ptr{Cvoid}, Int64, Int64, Ptr{Cvoid}, Ptr{Cvoid}),
                ctx.backend.handle, E, L, H, B, s4(x), s4(out), nullable(weight), weight === nothing ? 0 : dtcode(eltype(weight)),
                weight === nothing || ndims(weight) == 1 || size(weight, 2) == 1 ? 0 : stride(weight, 2), something(split, -1), eps,
                pointer(plan.freq), plan.rot, plan.interleaved, plan.gain, C_NULL, 0, 0, pointer(lens), nullable(news)))
    out
end

# kind 2: Int8, 3: e4m3 in UInt8 (b200dnn.h); k, v (E, T, H, P), kmax, vmax (H, P) Float32.
struct Cache8{K}
    k::K
    v::K
    kmax::B200Array{Float32,2}
    vmax::B200Array{Float32,2}
    kind::Int32
end
struct Cache8C                      # b200_cache8
    k::Ptr{Cvoid}
    v::Ptr{Cvoid}
    kstride::NTuple{4,Int64}
    vstride::NTuple{4,Int64}
    kmax::Ptr{Cvoid}
    vmax::Ptr{Cvoid}
    E::Int64
    T::Int64
    H::Int64
    P::Int64
    kind::Int32
    table::Ptr{Cvoid}
    table_ld::Int64
    width::Int64
end
cachec(c::Cache8, table) = Cache8C(s4(c.k).ptr, s4(c.v).ptr, s4(c.k).stride, s4(c.v).stride, pointer(c.kmax), pointer(c.vmax),
                                   size(c.k)..., c.kind, pointer(table), stride(table, 2), size(table, 1))

function cacheappend!(ctx::Ctx{B200Backend}, cache::Cache8, k, v, table, lens; news = nothing)
    check(ccall((:b200_cache_append, LIB), Cint,
                (Ptr{Cvoid}, Ref{Cache8C}, Int64, Int64, Ref{Strided4}, Ref{Strided4}, Ptr{Cvoid}, Ptr{Cvoid}),
                ctx.backend.handle, cachec(cache, table), size(k, 2), size(k, 4), s4(k), s4(v), pointer(lens), nullable(news)))
    cache
end
function cacheread!(ctx::Ctx{B200Backend}, out, cache::Cache8, values::Bool, table, lens; starts = nothing)
    check(ccall((:b200_cache_read, LIB), Cint,
                (Ptr{Cvoid}, Ref{Cache8C}, Cint, Int64, Int64, Ptr{Cvoid}, Ptr{Cvoid}, Ref{Strided4}, Cint),
                ctx.backend.handle, cachec(cache, table), values, size(out, 2), size(out, 4), nullable(starts), pointer(lens),
                s4(out), dtcode(eltype(out))))
    out
end
function cachesdpa!(ctx::Ctx{B200Backend}, out, q, cache::Cache8, table, lens; news = nothing, scale = 1 / sqrt(size(q, 1)), causal = true)
    check(ccall((:b200_cache_attention, LIB), Cint,
                (Ptr{Cvoid}, Ref{Cache8C}, Int64, Int64, Int64, Ref{Strided4}, Ref{Strided4}, Cint, Cfloat, Cint, Ptr{Cvoid}, Ptr{Cvoid}),
                ctx.backend.handle, cachec(cache, table), size(q, 2), size(q, 3), size(q, 4), s4(q), s4(out), dtcode(eltype(out)),
                Float32(scale), causal, pointer(lens), nullable(news)))
    out
end

s3(a) = (r = rootstrides(a); Strided4(Ptr{Cvoid}(r[1]), (Int64.(r[2])[1:3]..., Int64(0))))       # three axes
# Sequences side by side: q, out (E, N, Hq), k, v (E, Nk, H), starts and kstarts one Int32 more than sequences.
function packedsdpa!(ctx::Ctx{B200Backend}, out, q, k, v, starts; kstarts = starts, scale = 1 / sqrt(size(q, 1)), causal = true)
    demand(ndims(q) == ndims(k) == 3 && size(out) == size(q) && size(v) == size(k) && size(k, 1) == size(q, 1), "packedsdpa!: q and out are (E, N, Hq), k and v (E, Nk, H)")
    demand(eltype(q) === eltype(k) === eltype(v) === Float16 && eltype(out) in (Float16, Float32), "packedsdpa!: q, k and v are Float16")
    demand(length(starts) >= 1 && iscounts(starts, length(starts)) && kstarts !== nothing && iscounts(kstarts, length(starts)),
           "packedsdpa!: starts and kstarts are one Int32 more than sequences")
    demand(kstarts !== starts || size(k, 2) >= size(q, 2), "packedsdpa!: as many keys as rows where they lie at the same places")
    check(ccall((:b200_attention_packed_f16, LIB), Cint,
                (Ptr{Cvoid}, Int64, Int64, Int64, Int64, Int64, Int64, Ref{Strided4}, Ref{Strided4}, Ref{Strided4}, Ref{Strided4}, Cint, Cfloat, Cint,
                 Ptr{Cvoid}, Ptr{Cvoid}),
                ctx.backend.handle, size(q, 1), size(q, 2), size(k, 2), size(q, 3), size(k, 3), length(starts) - 1, s3(q), s3(k), s3(v), s3(out),
                dtcode(eltype(out)), Float32(scale), causal, pointer(starts), pointer(kstarts)))
    out
end

# The N best of K * V continuations: best, parents, tokens (N, B); logits (V, K, B), scores (K, B).
function beamselect!(ctx::Ctx{B200Backend}, best, parents, tokens, logits, scores; ended = nothing, pad = 0)
    demand(ndims(logits) == 3 && eltype(logits) in (Float16, Float32) && along(logits), "beamselect!: logits are (V, K, B) of Float16 or Float32")
    V, K, B = size(logits)
    demand(isdense(scores, Float32, K, B) && (ended === nothing || isdense(ended, Int32, K, B)), "beamselect!: scores and ended are dense (K, B)")
    demand(isdense(best, Float32, size(best, 1), B) && isdense(parents, Int32, size(best)...) && isdense(tokens, Int32, size(best)...),
           "beamselect!: best, parents and tokens are dense (N, B)")
    check(ccall((:b200_beam_select, LIB), Cint,
                (Ptr{Cvoid}, Int64, Int64, Int64, Int64, Ptr{Cvoid}, Cint, Int64, Int64, Ptr{Cvoid}, Ptr{Cvoid}, Int64, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}),
                ctx.backend.handle, V, K, B, size(best, 1), pointer(logits), dtcode(eltype(logits)), stride(logits, 2), stride(logits, 3),
                pointer(scores), nullable(ended), pad, pointer(best), pointer(parents), pointer(tokens)))
    best, parents, tokens
end

# Beam k of search b goes on from beam parents[k, b] (counted from 0) in all of `caches`; table, own (pages a sequence, K * B).
function cachereorder!(ctx::Ctx{B200Backend}, caches::AbstractVector, table, own, parents, lens)
    demand(ndims(parents) == 2 && isdense(parents, Int32, size(parents)...), "cachereorder!: parents are a dense (K, B) of Int32")
    demand(ndims(table) == 2 && eltype(table) === eltype(own) === Int32 && size(own) == size(table) && size(table, 2) == length(parents) && along(table) && along(own),
           "cachereorder!: table and own are (pages, K * B) of Int32")
    demand(lens !== nothing && iscounts(lens, length(parents)), "cachereorder!: lens is one Int32 a beam")
    demand(all(x -> size(x.v) == size(x.k) && size(x.kmax) == size(x.vmax) == size(x.k)[3:4], caches), "cachereorder!: caches are (E, T, H, P), their maxima (H, P)")
    c = Cache8C[cachec(x, table) for x in caches]
    check(ccall((:b200_cache_reorder, LIB), Cint,
                (Ptr{Cvoid}, Ptr{Cache8C}, Int64, Int64, Int64, Ptr{Cvoid}, Int64, Ptr{Cvoid}, Int64, Int64, Ptr{Cvoid}, Ptr{Cvoid}),
                ctx.backend.handle, c, length(c), size(parents, 1), size(parents, 2), pointer(table), stride(table, 2), pointer(own),
                stride(own, 2), size(table, 1), pointer(parents), pointer(lens)))
    table
end

struct Q4                           # b200_q4; the arrays it points to are Weight4's
    data::Ptr{Cvoid}
    scales::Ptr{Cvoid}
    zeros::Ptr{Cvoid}
    M::Int64
    K::Int64
    group::Int64
end
struct Weight4
    arrays::Tuple
    q4::Q4
end
# q (M, K) UInt8 of 0..15, scales (M, K ÷ group) Float16, zeros (M, K ÷ group) UInt8 or nothing
function pack4(ctx::Ctx{B200Backend}, q, scales, zeros; group = 64)
    M, K = size(q)
    n = ntuple(_ -> Ref{Int64}(0), 3)
    check(ccall((:b200_q4_sizes, LIB), Cint, (Int64, Int64, Int64, Ref{Int64}, Ref{Int64}, Ref{Int64}), M, K, group, n...))
    arrays = ntuple(i -> i == 3 && zeros === nothing ? nothing : KernelAbstractions.allocate(ctx.backend, UInt8, n[i][]), 3)
    w = Q4(nullable.(arrays)..., M, K, group)
    zst = zeros === nothing ? (0, 0) : strides(zeros)
    check(ccall((:b200_q4_pack, LIB), Cint,
                (Ptr{Cvoid}, Ptr{Cvoid}, Int64, Int64, Ptr{Cvoid}, Int64, Int64, Ptr{Cvoid}, Int64, Int64, Ref{Q4}),
                ctx.backend.handle, pointer(q), strides(q)..., pointer(scales), strides(scales)..., nullable(zeros), zst..., w))
    Weight4(arrays, w)
end
function matmul4!(ctx::Ctx{B200Backend}, out, W::Weight4, B, bias, epi)
    check(ccall((:b200_matmul_q4, LIB), Cint,
                (Ptr{Cvoid}, Ref{Q4}, Int64, Ptr{Cvoid}, Int64, Ptr{Cvoid}, Ptr{Cvoid}, Int64, Cint, Cint),
                ctx.backend.handle, W.q4, size(B, 2), pointer(B), stride(B, 2), nullable(bias), pointer(out), stride(out, 2),
                dtcode(eltype(out)), epicode(epi)))
    out
end

# ------------------------------------------------------------------ maxpool2d!, _to_copy (resample.jl:141, ops.jl:342-358)
function maxpool2d!(ctx::Ctx{B200Backend}, out, x, k, s, p)
    xs, os = rootstrides(x), rootstrides(out)     # any (x, y, c, n) view: the NCHW permutes need no copy
    W, H, C, N = size(x)
    check(ccall((:b200_maxpool2d_f16, LIB), Cint,
                (Ptr{Cvoid}, Int64, Int64, Int64, Int64, Ptr{Cvoid}, Ptr{Int64}, Ptr{Cvoid}, Ptr{Int64}, Int64, Int64, Int64,
                 Int64, Int64, Int64),
                ctx.backend.handle, W, H, C, N, Ptr{Cvoid}(xs[1]), collect(Int64.(xs[2])), Ptr{Cvoid}(os[1]),
                collect(Int64.(os[2])), k[1], k[2], s[1], s[2], p[1], p[2]))
    out
end
function tocopy!(ctx::Ctx{B200Backend}, out, a)
    check(ccall((:b200_cast, LIB), Cint, (Ptr{Cvoid}, Ptr{Cvoid}, Cint, Ptr{Cvoid}, Cint, Int64),
                ctx.backend.handle, pointer(a), dtcode(eltype(a)), pointer(out), dtcode(eltype(out)), length(a)))
    out
end

# ------------------------------------------------------------------ capture / replay! (SAM2Runner/src/sam2.jl:90-115)
# Run the ops once (sizes the pool and the workspace), then record them; replay! launches the graph.
function capture(f, b::B200Backend)
    f(); KernelAbstractions.synchronize(b)
    check(ccall((:b200_graph_begin, LIB), Cint, (Ptr{Cvoid},), b.handle))
    f()
    g = Ref{Ptr{Cvoid}}(C_NULL)
    check(ccall((:b200_graph_end, LIB), Cint, (Ptr{Cvoid}, Ref{Ptr{Cvoid}}), b.handle, g))
    g[]
end
replay!(b::B200Backend, g::Ptr{Cvoid}) = check(ccall((:b200_graph_launch, LIB), Cint, (Ptr{Cvoid}, Ptr{Cvoid}), b.handle, g))

# ------------------------------------------------------------------ convolution! (conv.jl:100-145)
function convolution!(ctx::Ctx{B200Backend}, out, x, w, bias, stride, padding, dilation, groups; act = :none)
    W, H, Cin, N = size(x); KW, KH, _, Cout = size(w)
    check(ccall((:b200_conv2d_grouped_f16, LIB), Cint,
                (Ptr{Cvoid}, Int64, Int64, Int64, Int64, Int64, Int64, Int64, Int64, Int64, Int64, Int64, Int64,
                 Int64, Int64, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Cint, Cint),
                ctx.backend.handle, W, H, Cin, N, KW, KH, Cout, stride[1], stride[2], padding[1], padding[2],
                dilation[1], dilation[2], groups, pointer(x), pointer(w), bias === nothing ? C_NULL : pointer(bias),
                pointer(out), dtcode(eltype(out)), act === :relu ? 1 : act === :gelu ? 2 : 0))
    out
end

# ------------------------------------------------------------------ convolutiontranspose! (conv.jl:247-290)
# shufflecase (stride == kernel, nothing else set, one group) runs as a GEMM + depth-to-space inside the
# library; every other geometry as the deterministic gather.  w is (KW, KH, Cout ÷ groups, Cin).
function convolutiontranspose!(ctx::Ctx{B200Backend}, out, x, w, bias, stride, padding, dilation, outpad, groups)
    W, H, Cin, N = size(x); KW, KH, Cog, _ = size(w)
    check(ccall((:b200_convtranspose2d_f16, LIB), Cint,
                (Ptr{Cvoid}, Int64, Int64, Int64, Int64, Int64, Int64, Int64, Int64, Int64, Int64, Int64, Int64,
                 Int64, Int64, Int64, Int64, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Cint),
                ctx.backend.handle, W, H, Cin, N, KW, KH, Cog * groups, stride[1], stride[2], padding[1], padding[2],
                dilation[1], dilation[2], outpad[1], outpad[2], groups, pointer(x), pointer(w),
                bias === nothing ? C_NULL : pointer(bias), pointer(out), dtcode(eltype(out))))
    out
end

# ------------------------------------------------------------------ Diagnostics (context.jl:162-221)
# optimes: bracket an op with the context's event timer (milliseconds on the device).
function optime(f, b::B200Backend)
    check(ccall((:b200_timer_start, LIB), Cint, (Ptr{Cvoid},), b.handle))
    f()
    ms = Ref{Cfloat}(0)
    check(ccall((:b200_timer_stop, LIB), Cint, (Ptr{Cvoid}, Ref{Cfloat}), b.handle, ms))
    Float64(ms[])
end
launchcount(b::B200Backend) = ccall((:b200_launch_count, LIB), Int64, (Ptr{Cvoid},), b.handle)

end # module
